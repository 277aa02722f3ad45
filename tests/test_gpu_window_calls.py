"""The windowed calls as programs make them: in HIP graphs, on other streams,
two at once, over large pools, with any workspace contents, and through the pager."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from strataflow_amd import _lib
from strataflow_amd.paged_kv import SFA_KV_F16, SFA_KV_F32, SFA_KV_Q8_0, PagedKV, rope_desc
from strataflow_amd.pager import SFA_ATTEND_WINDOW, KvPager

from .test_gpu_window import cuda, rows_of
from .window_ref import Cache, check, norm_rope

pytestmark = pytest.mark.gpu
F32, F16, Q8 = SFA_KV_F32, SFA_KV_F16, SFA_KV_Q8_0
TYPES = [F32, F16, Q8]


def lens_of(c):
    return torch.tensor(c.lens, dtype=torch.int32).cuda()


@pytest.mark.parametrize("kv_type", TYPES)
def test_graph_replays(gpu, kv_type):
    """Append, decode and prefill (split and not) captured, replayed with other inputs and eager work in between."""
    c = Cache(lens=[3000, 1700], n_head=8, n_head_kv=2, head_dim=128, page_size=256, kv_type=kv_type, seed=1)
    kv, rope = c.kv, rope_desc(128, 1e4, neox=True)
    lens, table = lens_of(c), c.t_table
    x = torch.empty(2, 12, 128).cuda()
    qc, ql = torch.empty(40, 8, 128).cuda(), torch.empty(1500, 8, 128).cuda()
    seq, pos = torch.arange(2, dtype=torch.int32).cuda(), lens - 1

    def step():
        q = kv.norm_rope_append(0, x[:, :8], x[:, 8:10], x[:, 10:], seq, pos, table, rope, q_norm=x.new_ones(128))
        return (q, kv.decode_window(0, q, table, lens, 3000, 1000, 4), kv.prefill_window(0, qc, table[0], 2960, 2000, 4),
                kv.prefill_window(0, ql, table[1], 200, 300, 4))

    x.normal_(), qc.normal_(), ql.normal_()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for seed in range(4):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (x, qc, ql):
            t.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        pools = kv.k.clone(), kv.v.clone()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(pools[0], kv.k) and torch.equal(pools[1], kv.v)


@pytest.mark.parametrize("kv_type", TYPES)
def test_the_same_call_gives_the_same_bits(gpu, kv_type):
    c = Cache(lens=[4000, 900], n_head=8, n_head_kv=2, head_dim=128, page_size=256, kv_type=kv_type, seed=2)
    q, qc = cuda(c.queries(2)), cuda(c.queries(60))
    d = [c.kv.decode_window(0, q, c.t_table, lens_of(c), 4000, 3000, 4) for _ in range(4)]
    p = [c.kv.prefill_window(0, qc, c.t_table[0], 3940, 2500, 4) for _ in range(4)]
    assert all(torch.equal(d[0], t) for t in d) and all(torch.equal(p[0], t) for t in p)


@pytest.mark.parametrize("as_handle", [False, True])
def test_other_streams_and_two_calls_at_once(gpu, as_handle):
    c = Cache(lens=[4000], n_head=8, n_head_kv=2, head_dim=128, page_size=256, seed=3)
    qs = [cuda(c.queries(1)) for _ in range(2)]
    qc = [cuda(c.queries(50)) for _ in range(2)]
    want = [c.kv.decode_window(0, q, c.t_table, lens_of(c), 4000, 3000, 4) for q in qs]
    want += [c.kv.prefill_window(0, q, c.t_table[0], 3950, 2500, 4) for q in qc]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    lens = lens_of(c)
    torch.cuda.synchronize()
    for _ in range(10):
        got = [None] * 4
        for i, s in enumerate(streams):
            h = s.cuda_stream if as_handle else s
            got[i] = c.kv.decode_window(0, qs[i], c.t_table, lens, 4000, 3000, 4, stream=h)
            got[2 + i] = c.kv.prefill_window(0, qc[i], c.t_table[0], 3950, 2500, 4, stream=h)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kv_type", TYPES)
def test_any_workspace_contents(gpu, kv_type):
    """Through the C ABI, with a workspace full of NaN and records of other calls."""
    c = Cache(lens=[3000, 0, 70], n_head=8, n_head_kv=2, head_dim=128, page_size=256, kv_type=kv_type, seed=4)
    lib, d = _lib.load(), c.kv.desc(0)
    q, lens = cuda(c.queries(3)), lens_of(c)
    want = c.kv.decode_window(0, q, c.t_table, lens, 3000, 2000, 4)
    need = lib.sfa_decode_window_workspace_bytes(d, 3, 3000, 2000, 4)
    need_p = lib.sfa_prefill_window_workspace_bytes(d, 2900, 30, 2000, 4)
    assert need > 256 and need_p > 0
    qc = cuda(c.queries(30))
    want_p = c.kv.prefill_window(0, qc, c.t_table[0], 2900, 2000, 4)
    ws = torch.full((max(need, need_p),), 0xFF, dtype=torch.uint8).cuda()
    s = _lib.current_stream()
    for _ in range(2):
        out, out_p = torch.full_like(want, 7), torch.full_like(want_p, 7)
        assert lib.sfa_attn_decode_window(d, q.data_ptr(), out.data_ptr(), c.t_table.data_ptr(), c.t_table.shape[1], lens.data_ptr(),
                                          2000, 4, 3, 3000, 128 ** -0.5, ws.data_ptr(), need, s) == 0
        assert lib.sfa_attn_prefill_window(d, qc.data_ptr(), out_p.data_ptr(), c.t_table[0].data_ptr(), c.t_table.shape[1], 2900, 30,
                                           2000, 4, 128 ** -0.5, ws.data_ptr(), need_p, s) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out_p, want_p)


@pytest.mark.parametrize("kv_type", [F32, F16, Q8])
def test_pools_past_32_bit_offsets(gpu, kv_type):
    """Pages whose bytes lie past 4 GiB of their pool."""
    c = Cache(lens=[700], n_head=32, n_head_kv=8, head_dim=128, page_size=256, kv_type=kv_type, seed=5)
    q, qc = cuda(c.queries(1)), cuda(c.queries(40))
    want = c.kv.decode_window(0, q, c.t_table, lens_of(c), 700, 500, 4)
    want_p = c.kv.prefill_window(0, qc, c.t_table[0], 660, 500, 4)
    n = (5 << 30) // c.kv.page_bytes
    big = PagedKV(1, 32, 8, 128, kv_type, 256, n)
    table = torch.full_like(c.t_table, -1)
    for lp in range(c.table.shape[1]):
        at = n - 1 - 2 * lp
        assert at * big.page_bytes > 1 << 32
        big.k[0, at], big.v[0, at] = c.kv.k[0, c.table[0, lp]], c.kv.v[0, c.table[0, lp]]
        table[0, lp] = at
    assert torch.equal(big.decode_window(0, q, table, lens_of(c), 700, 500, 4), want)
    assert torch.equal(big.prefill_window(0, qc, table[0], 660, 500, 4), want_p)
    # and the append into one
    x = torch.randn(3, 48, 128, generator=torch.Generator().manual_seed(0)).cuda()
    args = (x[:, :32], x[:, 32:40], x[:, 40:], torch.zeros(3, dtype=torch.int32).cuda(), torch.arange(600, 603, dtype=torch.int32).cuda())
    rope = rope_desc(128, 1e4)
    assert torch.equal(big.norm_rope_append(0, *args, table, rope), c.kv.norm_rope_append(0, *args, c.t_table, rope))
    lp = 600 // 256
    assert torch.equal(big.k[0, int(table[0, lp])], c.kv.k[0, c.table[0, lp]])
    assert torch.equal(big.v[0, int(table[0, lp])], c.kv.v[0, c.table[0, lp]])


def test_refusals_of_the_wrappers(gpu):
    c = Cache(lens=[100], seed=6)
    q, lens = cuda(c.queries(1)), lens_of(c)
    for bad in (dict(q=q.cpu()), dict(lens=lens.long()), dict(table=c.t_table[0]), dict(table=c.t_table.cpu()), dict(out=q.new_empty(2, 512)),
                dict(q=q.double())):
        a = dict(q=q, table=c.t_table, lens=lens, out=None)
        a.update(bad)
        with pytest.raises(ValueError):
            c.kv.decode_window(0, a["q"], a["table"], a["lens"], 100, 50, 4, out=a["out"])
    with pytest.raises(_lib.SfaError):
        c.kv.decode_window(0, q, c.t_table, lens, 100, 0, 4)
    with pytest.raises(ValueError):
        c.kv.prefill_window(0, q, c.t_table, 99, 50, 4)
    with pytest.raises(_lib.SfaError):
        c.kv.prefill_window(0, q, c.t_table[0], -1, 50, 4)
    x = torch.zeros(1, 12, 64).cuda()
    one = torch.zeros(1, dtype=torch.int32).cuda()
    rope = rope_desc(64, 1e4, sections=(16, 16))
    ok = dict(q=x[:, :8], k=x[:, 8:10], v=x[:, 10:], seq=one, pos=one, table=c.t_table)
    for bad, more in ((dict(k=x[:, 8:10].cpu()), {}), (dict(k=x[:, 8:11]), {}), (dict(seq=one.long()), {}), (dict(pos=one.cpu()), {}),
                      (dict(table=c.t_table.long()), {}), ({}, dict(q_norm=torch.ones(32).cuda())), ({}, dict(k_norm=torch.ones(64))),
                      ({}, dict(rope_pos=torch.zeros(1, 1, dtype=torch.int32).cuda())), ({}, dict(q_out=torch.zeros(1, 8, 32).cuda())),
                      (dict(q=None), dict(q_out=torch.zeros(1, 8, 64).cuda()))):
        a = dict(ok, **bad)
        with pytest.raises(ValueError):
            c.kv.norm_rope_append(0, a["q"], a["k"], a["v"], a["seq"], a["pos"], a["table"], rope, **more)


def test_nothing_to_do(gpu):
    c = Cache(lens=[100], seed=7)
    i = torch.zeros(0, dtype=torch.int32).cuda()
    assert c.kv.decode_window(0, torch.zeros(0, 8, 64).cuda(), c.t_table[:0], i, 100, 50, 4).shape == (0, 512)
    assert c.kv.prefill_window(0, torch.zeros(0, 8, 64).cuda(), c.t_table[0], 5, 50, 4).shape == (0, 512)
    x = torch.zeros(0, 12, 64).cuda()
    assert c.kv.norm_rope_append(0, x[:, :8], x[:, 8:10], x[:, 10:], i, i, c.t_table, rope_desc(64, 1e4)).shape == (0, 8, 64)


# ---- the pager -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("window,n_sink", [(100, 5), (64, 0), (150, 70)])
def test_pager_with_sinks(gpu, kv_type, window, n_sink):
    """Ragged chunks and single tokens of three sequences, pages released as the window moves on: every row is
    what 64 bits give of what the sequence appended."""
    Hq, Hkv, hd, n_seq, n_ctx = 8, 2, 64, 3, 700
    rng = np.random.default_rng(window)
    pager = KvPager(n_layer=2, n_head=Hq, n_head_kv=Hkv, head_dim=hd, kv_type=kv_type, page_size=64, n_seq=n_seq, n_ctx=n_ctx,
                    window=window, attend=SFA_ATTEND_WINDOW, n_sink=n_sink, seed=3)
    # what is held of each position, kept in a cache of its own through the same append
    keep = PagedKV(1, Hq, Hkv, hd, kv_type, 64, n_seq * 11)
    table = np.arange(n_seq * 11, dtype=np.int32).reshape(n_seq, 11)
    rope = rope_desc(hd, 1e4, neox=True)
    w = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    used = np.zeros(n_seq, int)
    steps = [(64, 30, 1), (1, 1, 1), (64, 0, 17), (50, 64, 64), (1, 1, 1), (64, 64, 2), (33, 64, 64), (1, 1, 1), (64, 7, 64), (1, 1, 1),
             (64, 64, 64), (64, 64, 64), (1, 1, 1)]
    for n_tok in steps:
        assert pager.begin(n_tok) == 0
        n = sum(n_tok)
        seq = np.repeat(np.arange(n_seq), n_tok)
        pos = np.concatenate([np.arange(used[b], used[b] + n_tok[b]) for b in range(n_seq)])
        x = cuda(rng.standard_normal((n, Hq + 2 * Hkv, hd)).astype(np.float32))
        q = pager.norm_rope_append(1, x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], rope, q_norm=cuda(w[0]), k_norm=cuda(w[1]))
        out = pager.attend(1, q)
        keep.norm_rope_append(0, None, x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], cuda(seq.astype(np.int32)), cuda(pos.astype(np.int32)), cuda(table),
                              rope, k_norm=cuda(w[1]))
        torch.cuda.synchronize()
        used += n_tok
        want, bound = [], []
        for b in range(n_seq):
            if n_tok[b] == 0:
                continue
            c = Cache.__new__(Cache)
            at = np.arange(used[b])
            c.Hq, c.Hkv, c.hd, c.ps, c.table, c.gone = Hq, Hkv, hd, 64, table, [np.zeros(704, bool)] * n_seq
            c.k = [rows_of(keep, keep.k, np.full(used[b], b), at, table)] * n_seq
            c.v = [rows_of(keep, keep.v, np.full(used[b], b), at, table)] * n_seq
            mine = np.nonzero(seq == b)[0]
            a, e = c.attend(b, q.cpu().numpy()[mine], pos[mine], window, n_sink)
            want.append(a)
            bound.append(e)
        check(out, np.concatenate(want), np.concatenate(bound), hd)
        assert pager.stats()["dev_pages_in_use"] <= n_seq * ((window + 62) // 64 + 2 + (n_sink + 63) // 64)
    assert pager.stats()["pages_dropped"] > 0
    pager.reset(1)
    assert pager.begin((0, 5, 0)) == 0
    pager.close()


def test_pager_append_attend_with_sinks(gpu):
    """The two calls in one give the two calls' bits."""
    outs = []
    for fused in (False, True):
        g = torch.Generator(device="cuda").manual_seed(0)
        pager = KvPager(n_layer=1, n_head=8, n_head_kv=2, head_dim=64, kv_type=F16, page_size=64, n_seq=2, n_ctx=512, window=70,
                        attend=SFA_ATTEND_WINDOW, n_sink=4)
        for n_tok in ((60, 64), (1, 1), (9, 0), (1, 1)):
            assert pager.begin(n_tok) == 0
            n = sum(n_tok)
            q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda") for h in (8, 2, 2))
            if fused:
                outs.append(pager.append_attend(0, k, v, q))
            else:
                pager.append(0, k, v)
                outs.append(pager.attend(0, q))
        torch.cuda.synchronize()
        pager.close()
    for a, b in zip(outs[:4], outs[4:]):
        assert torch.equal(a, b)
