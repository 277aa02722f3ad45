"""Window + sinks attention and the normed, rotated append on the GPU against
64-bit references, at the sizes, masks and layouts where they can go wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from strataflow_amd import _lib
from strataflow_amd.paged_kv import SFA_KV_F16, SFA_KV_F32, SFA_KV_Q8_0, PagedKV, rope_desc, row_bytes

from .window_ref import EPS24, Cache, check, decode_rows, norm_rope

pytestmark = pytest.mark.gpu
F32, F16, Q8 = SFA_KV_F32, SFA_KV_F16, SFA_KV_Q8_0
HEADS = {1: (3, 3), 2: (8, 4), 4: (32, 8), 8: (16, 2)}


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- decode -------------------------------------------------------------------------------------------

def run_decode(c, window, n_sink, q=None, max_seq_len=None, **kw):
    q = c.queries(len(c.lens)) if q is None else q
    out = c.kv.decode_window(0, cuda(q), c.t_table, torch.tensor(c.lens, dtype=torch.int32).cuda(),
                             max_seq_len or max(max(c.lens), 1), window, n_sink, **kw)
    torch.cuda.synchronize()
    want = [c.attend(b, q[b:b + 1], [n - 1], window, n_sink) for b, n in enumerate(c.lens)]
    check(out, np.concatenate([w for w, _ in want]), np.concatenate([e for _, e in want]), c.hd)
    return out


def seen_by_last(lens, window, n_sink):
    return lambda b, p: (p < n_sink) | (p > lens[b] - 1 - window)


@pytest.mark.parametrize("kv_type,hd", [(F32, 32), (F32, 64), (F32, 128), (F16, 32), (F16, 64), (F16, 128), (Q8, 64), (Q8, 128)])
@pytest.mark.parametrize("g", [1, 2, 4, 8])
def test_decode_types_and_heads(gpu, kv_type, hd, g):
    lens = [1, 2, 31, 32, 33, 64, 100, 129, 257, 700, 1500]
    Hq, Hkv = HEADS[g]
    c = Cache(lens=lens, there=seen_by_last(lens, 100, 5), n_head=Hq, n_head_kv=Hkv, head_dim=hd, kv_type=kv_type, seed=g)
    run_decode(c, 100, 5)


@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (1, 64), (2, 31), (32, 32), (33, 33), (63, 4), (64, 65), (65, 0),
                                           (500, 129), (1000, 1), (4096, 4), (2**31 - 1, 0), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("page_size", [32, 96, 256])
def test_decode_windows(gpu, window, n_sink, page_size):
    lens = [0, 1, 64, 65, 97, 1023, 2100]
    c = Cache(lens=lens, there=seen_by_last(lens, window, n_sink), page_size=page_size, seed=window % 1000 + n_sink % 1000)
    out = run_decode(c, window, n_sink)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_decode_long_and_wide(gpu, kv_type):
    lens = [9000, 5121, 1, 0, 12288, 7777]
    c = Cache(lens=lens, there=seen_by_last(lens, 4096, 4), n_head=32, n_head_kv=8, head_dim=128, page_size=256,
              kv_type=kv_type, seed=3)
    run_decode(c, 4096, 4)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_decode_one_long(gpu, kv_type):
    """The whole of a long sequence, split over the chip and joined."""
    c = Cache(lens=[20011], n_head=8, n_head_kv=2, head_dim=128, page_size=256, kv_type=kv_type, seed=4)
    run_decode(c, 2**31 - 1, 0)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_decode_many_sequences(gpu, kv_type):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 400, 150)]
    c = Cache(lens=lens, there=seen_by_last(lens, 200, 3), kv_type=kv_type, seed=5)
    run_decode(c, 200, 3)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_decode_cold_and_missing_pages(gpu, kv_type):
    c = Cache(lens=[1000, 300, 64], kv_type=kv_type, cold=9, seed=6, drop={(0, 3), (0, 15), (1, 0), (2, 0)})
    out = run_decode(c, 700, 130)
    assert (out[2] == 0).all()  # its only page is not there


@pytest.mark.parametrize("kv_type", [F32, F16])
def test_decode_peaks(gpu, kv_type):
    """Keys that raise the running maximum late, and scores far apart."""
    c = Cache(lens=[1500, 800], kv_type=kv_type, seed=7, boost=(97, 12.0))
    run_decode(c, 1200, 4)


def test_decode_past_the_table(gpu):
    """Positions past the table are not attended; a bound below the lengths still attends all of them."""
    c = Cache(lens=[640, 500], seed=8)
    q = c.queries(2)
    want = [c.attend(0, q[:1], [699], 300, 4), c.attend(1, q[1:], [499], 300, 4)]
    out = c.kv.decode_window(0, cuda(q), c.t_table, torch.tensor([700, 500], dtype=torch.int32).cuda(), 64, 300, 4)
    check(out, np.concatenate([w for w, _ in want]), np.concatenate([e for _, e in want]), c.hd)
    out = c.kv.decode_window(0, cuda(q), c.t_table, torch.tensor([2**31 - 1, -5], dtype=torch.int32).cuda(), 64, 300, 0)
    assert (out == 0).all()


def test_decode_bad_page_ids(gpu):
    """Ids outside the pools are as pages that are not there."""
    c = Cache(lens=[400], seed=9)
    c.table[0, 2], c.table[0, 4] = 10**6, -(10**6)
    c.gone[0] = np.repeat(np.isin(np.arange(c.table.shape[1]), (2, 4)), c.ps)
    c.t_table = cuda(c.table)
    run_decode(c, 350, 2)


def test_decode_queries_of_any_size(gpu):
    """Queries past 16 bits and very small ones: the scale takes them back."""
    c = Cache(lens=[300], seed=10)
    for f in (1e6, 1e-6):
        q = c.queries(1) * np.float32(f)
        out = c.kv.decode_window(0, cuda(q), c.t_table, torch.tensor([300], dtype=torch.int32).cuda(), 300, 200, 4,
                                 scale=0.125 / f)
        want, bound = c.attend(0, q, [299], 200, 4, scale=0.125 / f)
        check(out, want, bound, c.hd)


# ---- prefill --------------------------------------------------------------------------------------------

def run_prefill(c, past, window, n_sink):
    T = c.lens[0] - past
    q = c.queries(T)
    out = c.kv.prefill_window(0, cuda(q), c.t_table[0], past, window, n_sink)
    torch.cuda.synchronize()
    want, bound = c.attend(0, q, np.arange(past, past + T), window, n_sink)
    check(out, want, bound, c.hd)
    return out


def seen_by_chunk(past, window, n_sink):
    return lambda b, p: (p < n_sink) | (p > past - window)


@pytest.mark.parametrize("kv_type,hd", [(F32, 32), (F32, 64), (F32, 128), (F16, 32), (F16, 64), (F16, 128), (Q8, 64), (Q8, 128)])
@pytest.mark.parametrize("g", [1, 2, 4, 8])
def test_prefill_types_and_heads(gpu, kv_type, hd, g):
    Hq, Hkv = HEADS[g]
    past, T, W, ns = 333, 150, 100, 5
    c = Cache(lens=[past + T], there=seen_by_chunk(past, W, ns), n_head=Hq, n_head_kv=Hkv, head_dim=hd, kv_type=kv_type, seed=g)
    run_prefill(c, past, W, ns)


@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (2, 31), (64, 64), (63, 4), (65, 129), (130, 0), (500, 70),
                                           (2**31 - 1, 0), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("past,T", [(0, 1), (0, 64), (0, 300), (63, 2), (700, 1), (701, 33), (640, 257)])
def test_prefill_windows(gpu, window, n_sink, past, T):
    c = Cache(lens=[past + T], there=seen_by_chunk(past, window, n_sink), n_head=8, n_head_kv=2, seed=past + T)
    run_prefill(c, past, window, n_sink)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("T", [1, 3, 93, 700])
def test_prefill_on_a_long_past(gpu, kv_type, T):
    past = 9000
    c = Cache(lens=[past + T], there=seen_by_chunk(past, 2048, 4), n_head=8, n_head_kv=2, head_dim=128, page_size=256,
              kv_type=kv_type, seed=T)
    run_prefill(c, past, 2048, 4)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_prefill_cold_and_missing_pages(gpu, kv_type):
    c = Cache(lens=[900], kv_type=kv_type, cold=6, seed=6, drop={(0, 0), (0, 8), (0, 12)})
    out = run_prefill(c, 700, 40, 30)
    assert (out[768 + 39 - 700:832 - 700] == 0).all()  # their window's page and the sinks' are not there


def test_prefill_all_pages_missing(gpu):
    c = Cache(lens=[200], seed=6, drop={(0, lp) for lp in range(4)})
    assert (run_prefill(c, 100, 90, 4) == 0).all()


@pytest.mark.parametrize("kv_type", [F32, F16])
def test_prefill_peaks(gpu, kv_type):
    c = Cache(lens=[1100], kv_type=kv_type, seed=7, boost=(97, 12.0))
    run_prefill(c, 700, 512, 4)


@pytest.mark.parametrize("kv_type,hd", [(F32, 64), (F16, 64), (Q8, 64), (Q8, 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("past,T", [(0, 40), (200, 300)])
def test_prefill_masked_values_have_no_part(gpu, kv_type, hd, bad, past, T):
    """A row whose K and V are not finite: tokens that may not see it are as without it, the others NaN."""
    W, at = 50, past + T // 2
    c = Cache(lens=[past + T], kv_type=kv_type, head_dim=hd, seed=11)
    dt = torch.float32 if kv_type == F32 else torch.float16
    page = int(c.table[0, at // c.ps])
    for pool in (c.kv.k, c.kv.v):
        rows = pool[0, page].view(c.ps, c.Hkv, -1)[at % c.ps]
        if kv_type == Q8:
            rows = rows.view(c.Hkv, hd // 32, 34)[..., :2]  # the blocks' scales
            rows.copy_(torch.full((1,), bad, dtype=dt).cuda().view(torch.uint8).expand_as(rows))
        else:
            rows.copy_(torch.full((1, hd), bad, dtype=dt).cuda().view(torch.uint8).expand_as(rows))
    q = c.queries(T)
    out = c.kv.prefill_window(0, cuda(q), c.t_table[0], past, W, 3)
    t = np.arange(past, past + T)
    free = (t < at) | (t >= at + W)
    want, bound = c.attend(0, q, t, W, 3)
    check(out[torch.from_numpy(free).cuda()], want[free], bound[free], c.hd)
    assert torch.isnan(out[torch.from_numpy(~free).cuda()]).all()


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_prefill_masked_values_alone(gpu, kv_type, bad):
    """V alone not finite: the dims that it has of the rows that see it are not finite, nothing else is."""
    past, T, W, at = 100, 120, 50, 150
    c = Cache(lens=[past + T], kv_type=kv_type, head_dim=64, seed=12)
    dt = torch.float32 if kv_type == F32 else torch.float16
    rows = c.kv.v[0, int(c.table[0, at // c.ps])].view(c.ps, c.Hkv, -1)[at % c.ps]
    dims = np.zeros(64, bool)
    dims[32 if kv_type == Q8 else 37] = True
    if kv_type == Q8:
        dims[32:] = True
        rows.view(c.Hkv, 2, 34)[0, 1, :2] = torch.full((1,), bad, dtype=dt).cuda().view(torch.uint8)
    else:
        rows.view(dt)[0, 37] = bad
    q = c.queries(T)
    out = c.kv.prefill_window(0, cuda(q), c.t_table[0], past, W, 3)
    t = np.arange(past, past + T)
    want, bound = c.attend(0, q, t, W, 3)
    hit = np.zeros((T, c.Hq, 64), bool)
    hit[(t >= at) & (t < at + W), :c.Hq // c.Hkv] = dims
    hit = hit.reshape(T, -1)
    out = out.cpu().numpy()
    assert not np.isfinite(out[hit]).any()
    off = np.abs(np.where(hit, want, out) - want)
    assert (off <= bound).all()


# ---- append ----------------------------------------------------------------------------------------------

def rows_of(kv, pool, seq, pos, table):
    rb = row_bytes(kv.kv_type, kv.head_dim)
    b = pool[0].cpu().numpy().reshape(kv.n_pages, kv.page_size, kv.n_head_kv, rb)
    return decode_rows(b[table[seq, pos // kv.page_size], pos % kv.page_size], kv.kv_type, kv.head_dim)


def check_rows(got, want, err, kv_type):
    """Stored rows: half a step of the cache's type besides the error of the values themselves."""
    if kv_type == F32:
        tol = err
    elif kv_type == F16:
        tol = err + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    else:
        # a value is off by half a step of its block, d = amax / 127 itself by half a step of f16
        amax = np.abs(want).reshape(*want.shape[:-1], -1, 32).max(-1, keepdims=True)
        amax = np.broadcast_to(amax, (*amax.shape[:-1], 32)).reshape(want.shape)
        tol = 1.01 * err + amax * (1 / 254 + 2.0 ** -11) * (1 + 1e-5) + 127 * 2.0 ** -25
    off = np.abs(got - want)
    assert (off <= tol).all(), np.max(off - tol)


def run_append(*, kv_type=F16, heads=(8, 2), hd=64, n=20, n_rot=None, neox=True, sections=None, interleaved=False, norms=(True, True),
               page_size=64, stacked=True, pos0=0, base=1e4, seed=0, eps=1e-6, in_place=False, with_q=True, size=1.0):
    rng = np.random.default_rng(seed)
    Hq, Hkv = heads
    n_rot = n_rot or hd
    mp = -(-(pos0 + n) // page_size)
    kv = PagedKV(1, Hq, Hkv, hd, kv_type, page_size, mp + 2)
    kv.k.fill_(0x5A)
    kv.v.fill_(0x5A)
    table = np.stack([rng.permutation(mp + 2)[:mp]]).astype(np.int32)
    qkv = (rng.standard_normal((n, Hq + 2 * Hkv, hd)) * size).astype(np.float32)
    qkv[0, :, ::3] = 0
    qw, kw = (1 + 0.3 * rng.standard_normal((2, hd))).astype(np.float32)
    qw, kw = (qw if norms[0] else None), (kw if norms[1] else None)
    pos = np.arange(pos0, pos0 + n).astype(np.int32)
    rp = rng.integers(-50, 5000, (len(sections), n)).astype(np.int32) if sections else None
    rope = rope_desc(hd, base, n_rot=n_rot, neox=neox, sections=sections, interleaved=interleaved)
    x = cuda(qkv)
    if stacked:
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    else:
        q, k, v = x[:, :Hq].contiguous(), x[:, Hq:Hq + Hkv].contiguous(), x[:, Hq + Hkv:].contiguous()
    src = q.clone() if in_place else q
    out = kv.norm_rope_append(0, src if with_q else None, k, v, torch.zeros(n, dtype=torch.int32).cuda(), cuda(pos), cuda(table),
                              rope, q_norm=None if qw is None else cuda(qw), k_norm=None if kw is None else cuda(kw),
                              eps=eps, rope_pos=None if rp is None else cuda(rp), q_out=src if in_place else None)
    torch.cuda.synchronize()
    at = np.stack([pos]) if rp is None else rp
    wq = norm_rope(qkv[:, :Hq], qw, eps, at, n_rot, base, neox, sections, interleaved)
    wk = norm_rope(qkv[:, Hq:Hq + Hkv], kw, eps, at, n_rot, base, neox, sections, interleaved)

    def err(w, x, normed):
        # the larger of a head's values bounds a pair's: the norm's sum, root and products are some
        # sqrt(hd) + 8 half steps, an angle's rounding 4, a rotation's products and sum 4
        steps = (np.sqrt(hd) + 16) if normed else 8
        return steps * EPS24 * 2 * np.abs(w).max(-1, keepdims=True) + 1e-38

    if with_q:
        assert (np.abs(out.cpu().numpy() - wq) <= err(wq, qkv, norms[0])).all()
    else:
        assert out is None
    assert torch.equal(x, cuda(qkv))  # inputs stay
    seq = np.zeros(n, np.int64)
    check_rows(rows_of(kv, kv.k, seq, pos, table), wk, err(wk, qkv, norms[1]), kv_type)
    wv = qkv[:, Hq + Hkv:].astype(np.float64)
    check_rows(rows_of(kv, kv.v, seq, pos, table), wv, np.zeros_like(wv) + np.abs(wv) * 2 * EPS24, kv_type)
    # rows that no token names are as they were
    for pool in (kv.k, kv.v):
        rows = pool[0].cpu().numpy().reshape(kv.n_pages, page_size, -1)
        named = np.zeros((kv.n_pages, page_size), bool)
        named[table[0][pos // page_size], pos % page_size] = True
        assert (rows[~named] == 0x5A).all()
    return kv


@pytest.mark.parametrize("kv_type,hd", [(F32, 32), (F32, 64), (F32, 128), (F16, 32), (F16, 64), (F16, 128), (Q8, 64), (Q8, 128)])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("norms", [(True, True), (False, False), (True, False)])
def test_append_types(gpu, kv_type, hd, neox, norms):
    run_append(kv_type=kv_type, hd=hd, neox=neox, norms=norms, seed=hd)


@pytest.mark.parametrize("hd,n_rot", [(32, 8), (64, 24), (64, 32), (128, 64), (128, 104), (128, 128)])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("kv_type", [F16, Q8])
def test_append_part_of_a_head(gpu, hd, n_rot, neox, kv_type):
    if kv_type == Q8 and hd < 64:
        kv_type = F32
    run_append(hd=hd, n_rot=n_rot, neox=neox, kv_type=kv_type, seed=n_rot)


@pytest.mark.parametrize("hd,sections,interleaved", [(128, (16, 24, 24), False), (128, (24, 20, 20), True), (64, (20, 12), False),
                                                     (64, (16, 16), True), (32, (4, 4, 4, 4), True), (32, (0, 9, 0, 7), False),
                                                     (128, (64, 0, 0), True), (128, (22, 21, 21), True)])
@pytest.mark.parametrize("neox", [True, False])
def test_append_axes(gpu, hd, sections, interleaved, neox):
    run_append(hd=hd, sections=sections, interleaved=interleaved, neox=neox, kv_type=F32, seed=len(sections))


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (32, 8), (64, 8), (16, 16)])
@pytest.mark.parametrize("n", [1, 7, 300])
def test_append_heads_and_counts(gpu, heads, n):
    run_append(heads=heads, n=n, hd=128, page_size=32, seed=n)


@pytest.mark.parametrize("kw", [dict(stacked=False), dict(in_place=True), dict(with_q=False), dict(pos0=100000, page_size=1024),
                                dict(eps=0.0, size=1e-15), dict(size=1e15), dict(base=1e6, pos0=4000)])
def test_append_forms(gpu, kw):
    run_append(kv_type=F32, **kw)


def test_append_far_positions(gpu):
    """Angles of positions whose turns leave few digits in 32 bits."""
    rng = np.random.default_rng(1)
    kv = PagedKV(1, 4, 2, 128, F32, 64, 2)
    x = rng.standard_normal((3, 8, 128)).astype(np.float32)
    rp = np.array([[16777213, 2000003, -7654321]], np.int32)
    t = cuda(x)
    q = kv.norm_rope_append(0, t[:, :4], t[:, 4:6], t[:, 6:], torch.zeros(3, dtype=torch.int32).cuda(),
                            torch.arange(3, dtype=torch.int32).cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda(),
                            rope_desc(128, 1e4), rope_pos=cuda(rp))
    want = norm_rope(x[:, :4], None, 0, rp, 128, 1e4, False)
    assert np.abs(q.cpu().numpy() - want).max() <= 16 * EPS24 * np.abs(want).max()


def test_append_skipped_tokens(gpu):
    """Padding (negative seq or pos) is left alone; a token whose page is not there has its Q rotated only."""
    kv = PagedKV(1, 4, 2, 64, F16, 64, 3)
    kv.k.fill_(0x11)
    x = torch.randn(6, 8, 64, generator=torch.Generator().manual_seed(0)).cuda()
    seq = torch.tensor([0, -1, 0, 1, 0, 1], dtype=torch.int32).cuda()
    pos = torch.tensor([3, 4, -2, 70, 500, 2], dtype=torch.int32).cuda()
    table = torch.tensor([[1, -1], [2, 10**6]], dtype=torch.int32).cuda()
    out = torch.full((6, 4, 64), 7.0).cuda()
    kv.norm_rope_append(0, x[:, :4], x[:, 4:6], x[:, 6:], seq, pos, table, rope_desc(64, 1e4), q_out=out)
    same = (out == 7.0).flatten(1).all(1).tolist()
    assert same == [False, True, True, False, False, False]
    rows = kv.k[0].view(3, 64, -1)
    written = (rows != 0x11).any(-1).nonzero().tolist()
    assert written == [[1, 3], [2, 2]]


def test_append_norm_and_append_equal_the_plain_append(gpu):
    """Without norms and rotation by position 0 the pools are sfa_kv_append's, bit for bit."""
    for kv_type in (F32, F16, Q8):
        g = torch.Generator().manual_seed(kv_type)
        x = torch.randn(9, 8, 64, generator=g).cuda()
        a, b = (PagedKV(1, 4, 2, 64, kv_type, 64, 2) for _ in range(2))
        seq, pos = torch.zeros(9, dtype=torch.int32).cuda(), torch.arange(30, 39, dtype=torch.int32).cuda()
        table = torch.tensor([[1]], dtype=torch.int32).cuda()
        a.norm_rope_append(0, None, x[:, 4:6], x[:, 6:], seq, pos, table, rope_desc(64, 1e4),
                           rope_pos=torch.zeros(1, 9, dtype=torch.int32).cuda())
        b.append(0, x[:, 4:6].contiguous(), x[:, 6:].contiguous(), seq, pos, table)
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


# ---- together ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_prompt_then_tokens(gpu, kv_type):
    """A prompt in chunks, then single tokens: what the attentions give is what 64 bits give of the rows held."""
    Hq, Hkv, hd, ps, W, ns = 8, 2, 64, 64, 90, 5
    rng = np.random.default_rng(2)
    kv = PagedKV(1, Hq, Hkv, hd, kv_type, ps, 12)
    table = rng.permutation(12)[:8].astype(np.int32)[None]
    rope = rope_desc(hd, 1e4, neox=True, sections=(12, 10, 10), interleaved=True)
    w = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    used, t_table = 0, cuda(table)
    for n in (150, 1, 70, 1, 1, 33, 1):
        x = cuda(rng.standard_normal((n, Hq + 2 * Hkv, hd)).astype(np.float32))
        pos = np.arange(used, used + n).astype(np.int32)
        rp = np.stack([pos, pos // 3, pos % 3]).astype(np.int32)
        q = kv.norm_rope_append(0, x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], torch.zeros(n, dtype=torch.int32).cuda(),
                                cuda(pos), t_table, rope, q_norm=cuda(w[0]), k_norm=cuda(w[1]), rope_pos=cuda(rp))
        used += n
        if n == 1:
            out = kv.decode_window(0, q, t_table, torch.tensor([used], dtype=torch.int32).cuda(), 512, W, ns)
        else:
            out = kv.prefill_window(0, q, t_table[0], used - n, W, ns)
        c = Cache.__new__(Cache)
        c.Hq, c.Hkv, c.hd, c.ps, c.table, c.gone = Hq, Hkv, hd, ps, table, [np.zeros(512, bool)]
        at = np.arange(used)
        c.k = [rows_of(kv, kv.k, np.zeros(used, np.int64), at, table)]
        c.v = [rows_of(kv, kv.v, np.zeros(used, np.int64), at, table)]
        want, bound = c.attend(0, q.cpu().numpy(), pos, W, ns)
        check(out, want, bound, hd)
