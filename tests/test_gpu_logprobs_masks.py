"""Log probabilities of rows masked with large finite logits (a type's lowest value, -1e38, -3e37) in place of -inf."""
import pytest
import torch

from ops_reference import TYPES
from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(4, 3000), (5, 151936), (1100, 20000)])
def test_entropy_under_finite_masks(gpu, rows, vocab, t):
    """Live ids at the ends, in one lane's piece, and spread, over a mask that fills whole tiles: lanes that have met masked logits
    alone go over to an ordinary maximum, within a part, among lanes, waves and parts."""
    g = torch.Generator().manual_seed(vocab)
    base = (torch.randn((rows, vocab), generator=g) * 2).to(TYPES[t])
    low = torch.finfo(TYPES[t]).min
    i = torch.arange(vocab)
    for mask in (low,) if t == "f16" else (low, -1e38, -3e37, -1e36):
        x = torch.full((rows, vocab), mask, dtype=TYPES[t])
        for r, live in enumerate((i >= vocab - 5, i < 7, (i >= vocab // 2) & (i < vocab // 2 + 16), i % 977 == 13)):
            x[r::4, live] = base[r::4, live]
        x = x.cuda()
        print(f"case masks {rows} x {vocab} {t} {mask:g}", flush=True)
        for top in (0, 4):
            r = check(x[:4] if rows > 100 else x, [vocab - 1, 0, vocab // 2, 13, vocab - 2][:min(rows, 5) if rows <= 100 else 4], top)
            assert torch.isfinite(r.entropy).all()
        if rows > 100:  # one block per row
            from zerollm_amd.ops import logprobs as own
            many = own(x)
            assert torch.isfinite(many.entropy).all()
            e = torch.stack([check(x[j:j + 1], None, 0).entropy[0] for j in range(0, rows, 97)])
            assert ((many.entropy[::97] - e).abs() <= 2 * (2.0 ** -19 + 2.0 ** -22 * 5 * 16)).all()


def test_rows_of_two_far_values(gpu):
    """Every logit at the lowest value but one; all at it; the mask after the live ones and before."""
    for t in (torch.float32, torch.bfloat16):
        x = torch.full((4, 9000), torch.finfo(t).min, dtype=t)
        x[0, 8999], x[1, 0] = 3.0, -2.0
        x[3, :4500] = torch.finfo(t).max
        r = check(x.cuda(), [8999, 0, 5, 1], 3)
        e = r.entropy.double().cpu()
        assert e[0] == 0 and e[1] == 0 and abs(e[2] - torch.tensor(9000.0).log()) < 1e-5 and abs(e[3] - torch.tensor(4500.0).log()) < 1e-5
