"""The windowed calls at the ends of their arguments' ranges: scales and
queries so small that their product is no f32, lengths at both ends of int32."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from strataflow_amd.paged_kv import SFA_KV_F16, SFA_KV_F32, SFA_KV_Q8_0

from .test_gpu_window import cuda
from .window_ref import Cache, check

pytestmark = pytest.mark.gpu
TYPES = [SFA_KV_F32, SFA_KV_F16, SFA_KV_Q8_0]
INT_MAX, INT_MIN = 2 ** 31 - 1, -2 ** 31


@pytest.mark.parametrize("scale", [1e-3, 1e-8, 1e-37])
@pytest.mark.parametrize("kv_type", TYPES)
def test_rows_of_zeros_attend_evenly(gpu, kv_type, scale):
    """A query of zeros under a small scale: the mean of the visible V, with masked and missing places beside them."""
    c = Cache(lens=[700], n_head=4, n_head_kv=2, head_dim=128, page_size=64, kv_type=kv_type, seed=5, drop={(0, 8)})
    q = np.zeros((1, 4, 128), np.float32)
    got = c.kv.decode_window(0, cuda(q), c.t_table, torch.tensor([700], dtype=torch.int32).cuda(), 700, 333, 3, scale=scale)
    check(got, *c.attend(0, q, [699], 333, 3, scale), 128)
    q = np.zeros((90, 4, 128), np.float32)
    q[::2] = c.queries(45) * 1e-30
    got = c.kv.prefill_window(0, cuda(q), c.t_table[0], 610, 333, 3, scale=scale)
    check(got, *c.attend(0, q, np.arange(610, 700), 333, 3, scale), 128)


@pytest.mark.parametrize("kv_type", TYPES)
def test_lengths_at_both_ends(gpu, kv_type):
    """A length under zero gives zeros whatever it is; the longest one attends what the table holds, over tables
    whose positions pass 31 bits."""
    c = Cache(lens=[100, 64, 64, 64], n_head=2, n_head_kv=2, head_dim=64, page_size=64, kv_type=kv_type, seed=6)
    q = c.queries(4)
    lens = torch.tensor([100, 0, -1, INT_MIN], dtype=torch.int32).cuda()
    got = c.kv.decode_window(0, cuda(q), c.t_table, lens, 100, INT_MAX, 0)
    check(got[:1], *c.attend(0, q[:1], [99], INT_MAX, 0), 64)
    assert not got[1:].any()

    table = torch.full((1, 2 ** 25 + 3), -1, dtype=torch.int32).cuda()
    table[0, :2] = c.t_table[0, :2]
    c.k[0], c.v[0] = c.k[0][:64], c.v[0][:64]
    lens = torch.tensor([INT_MAX], dtype=torch.int32).cuda()
    got = c.kv.decode_window(0, cuda(q[:1]), table, lens, INT_MAX, 1, 64)
    check(got, *c.attend(0, q[:1], [INT_MAX - 1], 1, 64), 64)
    got = c.kv.prefill_window(0, cuda(q), table[0], INT_MAX - 4, 2, 64)
    check(got, *c.attend(0, q, INT_MAX - 4 + np.arange(4), 2, 64), 64)
    # every position before the window a sink
    table[0, 1] = -1
    got = c.kv.decode_window(0, cuda(q[:1]), table, lens, INT_MAX, 1, INT_MAX)
    check(got, *c.attend(0, q[:1], [INT_MAX - 1], 1, INT_MAX), 64)


def test_arguments_past_32_bits(gpu):
    c = Cache(lens=[64], n_head=2, n_head_kv=2, head_dim=64, page_size=64, seed=7)
    q, lens = cuda(c.queries(1)), torch.tensor([64], dtype=torch.int32).cuda()
    for more in ((2 ** 32 + 64, 8, 0), (64, 2 ** 32 + 8, 0), (64, 8, 2 ** 31)):
        with pytest.raises(ValueError):
            c.kv.decode_window(0, q, c.t_table, lens, *more)
    for more in ((2 ** 32 + 63, 8, 0), (63, 2 ** 32 + 8, 0), (63, 8, 2 ** 31)):
        with pytest.raises(ValueError):
            c.kv.prefill_window(0, q, c.t_table[0], *more)
