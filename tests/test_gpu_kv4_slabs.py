"""Attention calls whose records do not fit the work space at once: run in slabs, in a bounded work space, with the same bits."""
import pytest
import torch

from ops_reference import TYPES
from test_gpu_kv4 import cache, ints, rows

pytestmark = pytest.mark.gpu

MOST = 2 ** 29


def test_work_space_is_bounded(gpu):
    """By capacity and rows: 2^29 bytes, or one token's where that is more; and no less for a part of a call's tokens' form."""
    c = cache(3, 8, 128, 131072)
    assert c.work_bytes(1, 256, 32) <= MOST
    for seqs, tokens, heads in ((1, 2048, 32), (1, 65536, 32), (3, 4000, 64), (65535, 1, 8), (1, 2 ** 21, 32)):
        assert MOST // 2 < c.work_bytes(seqs, tokens, heads) <= MOST
    c.close()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_long_prompts_in_slabs(gpu, t):
    """600 tokens of 32 heads in a cache of 131072 (1.3 GB of records as one): after a short and a long prefix, with a count, in place
    and in a work space of just the size, against 50 tokens at a time."""
    kv, H, D, n, T = 8, 32, 128, 20000, 600
    c = cache(1, kv, D, 131072)
    k, v = rows(1, (1, n, kv, D), "f16"), rows(2, (1, n, kv, D), "f16")
    c.append(k, v, ints(0))
    assert T * H * 128 * 520 > 2 * MOST
    work = torch.empty(c.work_bytes(1, T, H), dtype=torch.uint8, device="cuda")
    q = rows(3, (1, T, H, D), t, "head")
    for first in (-3, 0, n - T):
        want = torch.cat([c.attend(q[:, i:i + 50], ints(first + i)) for i in range(0, T, 50)], 1)
        print(f"case slabs at {first} {t}", flush=True)
        assert (c.attend(q, ints(first), work=work) == want).all()
        same = q.clone()
        c.attend(same, ints(first), out=same)
        assert (same == want).all()
        for count in (0, 200, 241, 599):
            out = torch.full_like(q, 5.0)
            c.attend(q, ints(first), count=ints(count), out=out, work=work)
            assert (out[:, :count] == want[:, :count]).all() and (out[:, count:] == 5.0).all()
    c.close()


@pytest.mark.parametrize("slots", [True, False])
def test_many_sequences_in_slabs(gpu, slots):
    """Sequences of 60 tokens each, ragged counts, each in its own slot or several in one, against one sequence at a time."""
    S, kv, H, D, T, cap = 300, 1, 8, 64, 60, 16384
    c = cache(7 if slots else S, kv, D, cap)
    assert S * T * H * (cap // 1024) * (D + 2) * 4 > MOST >= c.work_bytes(S, T, H)
    g = torch.Generator().manual_seed(5)
    slot = torch.randint(0, 9, (S,), generator=g).tolist() if slots else list(range(S))  # (7 and 8 do not exist)
    pos = torch.randint(0, 1500, (S,), generator=g).tolist()
    count = torch.randint(0, T + 3, (S,), generator=g).tolist()
    x = rows(6, (c.n_slot, 1600, kv, D), "f16")
    c.append(x, x, ints(*[0] * c.n_slot))
    q = rows(7, (S, T, H, D))
    out = torch.full_like(q, 5.0)
    print(f"case sequences slots {slots}", flush=True)
    c.attend(q, ints(*pos), count=ints(*count), slot=ints(*slot) if slots else None, out=out)
    for s in list(range(0, S, 7)) + [S - 1]:
        n = min(count[s], T)
        want = c.attend(q[s:s + 1], ints(pos[s]), slot=ints(slot[s]))
        same = (out[s, :n] == want[0, :n]) | (out[s, :n].isnan() & want[0, :n].isnan())
        assert same.all() and (out[s, n:] == 5.0).all(), s
    c.close()


def test_more_rows_than_a_grid_holds(gpu):
    """65535 sequences of 257 KV heads that share two slots: a block for each (sequence, head) would be 2^32 threads and more."""
    S, kv, D = 65535, 257, 64
    c = cache(2, kv, D, 64)
    k = rows(8, (2, 64, kv, D), "f16")
    c.append(k, k, ints(0, 0))
    pos = (torch.arange(S) % 60).int().cuda()
    slot = (torch.arange(S) % 2).int().cuda()
    q = torch.randn((S, 1, kv, D), device="cuda", dtype=TYPES["f16"])
    few = [0, 1, 2, 12345, 40000, S - 1]
    want = c.attend(q[few], pos[few], slot=slot[few])
    print("case grid", flush=True)
    c.attend(q, pos, slot=slot, out=q)
    assert (q[few] == want).all()
    c.close()
