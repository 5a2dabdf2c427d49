"""Rotary positions of very many tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_tokens_than_a_grid_holds_blocks(gpu):
    """2^24 tokens of a head so wide that a block takes one token: 2^32 threads at a block a token. 69 GB, in place."""
    from zerollm_amd.ops import Rope
    n, dim = 2 ** 24 + 5, 2050
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("needs 69 GB")
    r = Rope(2)
    q = torch.ones((1, n, 1, dim), dtype=torch.float16, device="cuda")
    pos = torch.tensor([7], dtype=torch.int32, device="cuda")
    few = [0, 1, 12345678, n - 2, n - 1]
    want = [r.apply(q[:, t:t + 1], None, pos + t)[0] for t in few]
    print("case many tokens", flush=True)
    r.apply(q, None, pos, out=(q, None))
    for t, w in zip(few, want):
        assert (q[:, t:t + 1] == w).all() and (w[..., 2:] == 1).all() and (w[..., :2] != 1).any(), t
    r.close()
