"""Appends of many sequences that share slots."""
import numpy as np
import pytest
import torch

from ops_reference import stored
from test_gpu_kv4 import cache, f64, ints, read, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,slots,tokens", [(700, 3, 5), (257, 300, 2), (65535, 64, 1), (1500, 1, 40)])
def test_sequences_of_one_slot_in_order(gpu, S, slots, tokens):
    """Far apart in the batch, in every wave's share of it, some of them dropped, overlapping: the last one's values stay. (A block used
    to walk all sequences one after the other, before its own and after: 65535 of them kept the GPU for seconds.)"""
    cap, dim = 200, 64
    c = cache(slots, 2, dim, cap)
    g = np.random.default_rng(S)
    slot, pos, count = g.integers(-1, slots + 1, S), g.integers(-3, cap + 1, S), g.integers(0, tokens + 2, S)
    few = rows(1, (1, 509, 2, dim))[0], rows(2, (1, 509, 2, dim))[0]  # (values from a table, by sequence and token)
    which = torch.from_numpy((np.arange(S)[:, None] * 7 + np.arange(tokens) * 3) % 509).cuda()
    print(f"case slots {S} {slots} {tokens}", flush=True)
    c.append(few[0][which], few[1][which], ints(*pos), ints(*count), ints(*slot))
    want = np.full((slots, cap), -1)
    w = which.cpu().numpy()
    for s in range(S):
        for j in range(min(tokens, count[s])):
            if 0 <= slot[s] < slots and 0 <= pos[s] + j < cap:
                want[slot[s], pos[s] + j] = w[s, j]
    got = np.stack(read(c, [0] * slots, cap))
    for x, table in zip(got, few):
        t = np.concatenate([stored(f64(table)), np.zeros((1, 2, dim))])  # (-1: never written)
        assert (x == t[want]).all()
    c.close()
