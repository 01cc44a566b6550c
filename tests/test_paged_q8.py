"""The paged cache in 8 bits (qd_paged_append_q8, qd_paged_read_q8, qd_paged_attn_decode_q8): refusals on the
host (no GPU), and the CUDA path against plain 64-bit evaluations.

Tolerances count roundings. Of the attention, relative to A = sum of |weight| |value| of an output:
 - scores: as in test_paged.py (f32 sums and q as two f16: S (2^-19 + 2^-21)), and the product with the query's factor
   and the row's scale: S 2^-22;
 - weights: twice that, 2^-20 for the exponential, 2^-21 for two f16 parts; V's scale goes in by its exponent, at
   most L + 1 in size for |log2 scale| <= L, whose sum with the score is off by 2^-24 (1.45 S + L + 1), and by its
   factor, off by 2^-24: together less than the 2^-22 L + 2^-24 (1.45 S + L) that a logarithm would cost, or, for
   L < 1, than what 2^-20 leaves over;
 - sums over n keys in f32: n / 16 * 2^-23 + 2^-19; the output's own rounding.
Of a row written in 8 bits: n is x / scale rounded, so |x - n scale| <= scale / 2 but for f32 roundings: of x itself
(its tolerance), of the scale and its inverse (2^-23 of 127 steps)."""
import math

import pytest

from kernel_optimization_webgpu_b200 import _lib
from test_paged import BASE, D, HALF_STEP, HEADS, LENS, _cuda, _kv, _refuses, _types, close, make_cache


# ---- refusals (no GPU) -----------------------------------------------------------------

def _q8(**kw):
    d = dict(k=4096, v=8192, k_scale=4096, v_scale=8192, num_pages=4, page_size=16, kv_heads=2, head_dim=128, batch=2,
             block_table=4096, table_width=3, table_stride=3, seq_lens=4096, status=None)
    d.update(kw)
    return _lib.QdPagedQ8(*(d[n] for n, _ in _lib.QdPagedQ8._fields_))


BAD = [dict(page_size=24), dict(page_size=8), dict(page_size=512), dict(head_dim=64), dict(kv_heads=0), dict(batch=-1),
       dict(batch=4097), dict(num_pages=-1), dict(table_stride=2), dict(block_table=None), dict(seq_lens=None), dict(k=None),
       dict(v=8200), dict(k_scale=None), dict(v_scale=None), dict(k_scale=4100), dict(table_width=1 << 27, table_stride=1 << 27)]


@pytest.mark.parametrize("bad", BAD, ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_a_bad_cache_is_refused_by_every_entry(bad):
    L = _lib.load()
    kv = _q8(**bad)
    calls = (lambda: L.qd_paged_append_q8(kv, BASE, 1, 768, 2, None, 2, None, None, 1e-6, None, None, 0, 0, BASE, 1, 768, None),
             lambda: L.qd_paged_attn_decode_q8(kv, BASE, 1, 256, 2, 0, 0, 0.0, 2 * BASE, 256, 4096, None),
             lambda: L.qd_paged_read_q8(kv, None, _kv(k=BASE, v=2 * BASE), None))
    for call in calls:
        assert call() == _lib.QD_E_INVALID
        assert L.qd_last_error(None).startswith(b"paged cache")
    for call in (lambda: L.qd_paged_append_q8(None, BASE, 1, 768, 2, None, 2, None, None, 1e-6, None, None, 0, 0, BASE, 1, 768, None),
                 lambda: L.qd_paged_attn_decode_q8(None, BASE, 1, 256, 2, 0, 0, 0.0, 2 * BASE, 256, 4096, None),
                 lambda: L.qd_paged_read_q8(None, None, _kv(), None), lambda: L.qd_paged_read_q8(_q8(), None, None, None)):
        assert call() == _lib.QD_E_INVALID


def test_attention_arguments_are_refused():
    L = _lib.load()
    ok = dict(q=BASE, dtype=1, stride=256, heads=2, window=0, sinks=0, scale=0.0, y=2 * BASE, y_stride=256, ws=4096)
    for bad in [dict(q=None), dict(y=None), dict(ws=None), dict(q=BASE + 8), dict(dtype=3), dict(dtype=-1), dict(stride=248),
                dict(stride=260), dict(y_stride=128), dict(heads=3), dict(heads=0), dict(heads=130, stride=130 * 128, y_stride=130 * 128),
                dict(window=-1), dict(sinks=-1), dict(scale=math.inf), dict(scale=math.nan), dict(ws=4104),
                dict(y=BASE), dict(y=4096), dict(y=8192 + 16)]:
        c = {**ok, **bad}
        rc = L.qd_paged_attn_decode_q8(_q8(), c["q"], c["dtype"], c["stride"], c["heads"], c["window"], c["sinks"], c["scale"],
                                       c["y"], c["y_stride"], c["ws"], None)
        assert rc == _lib.QD_E_INVALID, bad
    assert L.qd_paged_attn_decode_q8(_q8(batch=0), None, 1, 256, 2, 0, 0, 0.0, None, 256, None, None) == _lib.QD_OK
    kv = _q8(batch=4096, table_width=1 << 22, table_stride=1 << 22, block_table=64, seq_lens=64)
    assert L.qd_paged_attn_decode_q8(kv, BASE, 1, 256, 2, 0, 0, 0.0, 2 * BASE, 256, 4096, None) == _lib.QD_E_RANGE


def test_append_arguments_are_refused():
    L = _lib.load()
    ok = dict(qkv=BASE, dtype=1, stride=768, rows=2, heads=2, qn=None, eps=1e-6, cos=4096, sin=4096, rope_len=640,
              rope_stride=64, out=2 * BASE, out_dtype=1, out_stride=256)
    for bad in [dict(qkv=None), dict(out=None), dict(qkv=BASE + 4), dict(dtype=3), dict(out_dtype=-1), dict(stride=760),
                dict(rows=-1), dict(rows=3), dict(heads=-1), dict(eps=math.nan), dict(sin=None), dict(rope_stride=2),
                dict(out_stride=128), dict(qn=4100), dict(out=BASE + 256), dict(out=4096), dict(qkv=8192)]:
        c = {**ok, **bad}
        rc = L.qd_paged_append_q8(_q8(), c["qkv"], c["dtype"], c["stride"], c["rows"], None, c["heads"], c["qn"], None, c["eps"],
                                  c["cos"], c["sin"], c["rope_len"], c["rope_stride"], c["out"], c["out_dtype"],
                                  c["out_stride"], None)
        assert rc == _lib.QD_E_INVALID, bad
    assert L.qd_paged_append_q8(_q8(), None, 1, 768, 0, 4096, 2, None, None, 1e-6, None, None, 0, 0, None, 1, 256, None) == _lib.QD_OK


def test_read_arguments_are_refused():
    L = _lib.load()
    pools = dict(k=BASE, v=2 * BASE)
    for to in (_kv(**pools, batch=1), _kv(**pools, kv_heads=4), _kv(**pools, dtype=_lib.QD_KV_F32), _kv(**pools, head_dim=64),
               _kv(k=None, v=BASE), _kv(k=4096, v=BASE), _kv(k=BASE, v=4096 + 4 * 2 * 16 * 128 - 256)):
        assert L.qd_paged_read_q8(_q8(), None, to, None) == _lib.QD_E_INVALID
    assert _refuses(L.qd_paged_read_q8, _q8(batch=0), None, _kv(**pools, batch=0, seq_lens=None), None) == ""
    far = dict(batch=4096, table_width=1 << 22, table_stride=1 << 22)
    assert L.qd_paged_read_q8(_q8(**far), None, _kv(**pools, **far), None) == _lib.QD_E_RANGE


def test_python_wrappers_refuse_before_they_enqueue():
    torch = pytest.importorskip("torch")
    from kernel_optimization_webgpu_b200 import runtime as R
    k = torch.zeros(4, 2, 16, D, dtype=torch.int8)
    s = torch.zeros(4, 2, 16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 2, D)
    for args in ((q, k, k[:3], s, s, table, lens), (q, k.half(), k.half(), s, s, table, lens), (q, k, k, s[:3], s, table, lens),
                 (q, k, k, s, s.half(), table, lens), (q, k, k, s, s, table.long(), lens), (q[:1], k, k, s, s, table, lens),
                 (q, k, k, s, s, table, lens)):   # the last: not CUDA tensors
        with pytest.raises(ValueError):
            R.paged_attn_decode_q8(*args)
    out = torch.zeros(4, 2, 16, D, dtype=torch.float16)
    with pytest.raises(ValueError):
        R.paged_read_q8(k, k, s, s, table, lens, out, out, table)
    with pytest.raises(ValueError):
        R.paged_append_q8(torch.zeros(2, 700), k, k, s, s, table, lens, None, None, 2)


# ---- caches and plain forms ----------------------------------------------------------------

def make_q8(torch, totals, page, kv_heads, seed=0, fill=True, width=None, spread=4.0):
    """An 8-bit cache of random rows whose scales lie within 2^spread of each other either way, rows that no
    sequence holds with NaN scales; (k, v, ks, vs, table, lens)."""
    k, v, table, n = make_cache(torch, totals, page, kv_heads, "f16", seed=seed, fill=math.nan if fill else None, width=width)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    out = []
    for x in (k, v):
        scale = 2.0 ** ((torch.rand(x.shape[:3], generator=g, device="cuda") * 2 - 1) * spread) / 60
        ints = torch.randint(-127, 128, x.shape, generator=g, device="cuda").to(torch.int8)
        out += [ints, torch.where(x[..., 0].isnan(), math.nan, scale)]
    k8, ks, v8, vs = out
    return k8, v8, ks, vs, table, n


def plain(torch, q, k, v, ks, vs, table, lens, window, sinks, scale, io):
    """(y, tolerance) in 64 bits."""
    page, kvh, H = k.shape[2], k.shape[1], q.shape[1]
    ys, tols = [], []
    for b in range(q.shape[0]):
        t = max(int(lens[b]), 0)
        j = torch.arange(t, device="cuda")
        if window:
            j = j[(j > t - 1 - window) | (j < sinks)]
        if t == 0:
            ys.append(torch.zeros(H, D, device="cuda", dtype=torch.float64))
            tols.append(torch.full((H, D), 1e-30, device="cuda", dtype=torch.float64))
            continue
        pg = table[b].long()[j // page]
        kk, vv = (x[pg, :, j % page].double() * s[pg, :, j % page].double()[..., None] for x, s in ((k, ks), (v, vs)))
        kk, vv = (x.repeat_interleave(H // kvh, 1) for x in (kk, vv))
        qs = q[b].double()
        s = torch.einsum("hd,jhd->hj", qs, kk) * scale
        S = (torch.einsum("hd,jhd->hj", qs.abs(), kk.abs()) * abs(scale)).amax(-1)[:, None]
        w = torch.softmax(s, -1)
        y = torch.einsum("hj,jhd->hd", w, vv)
        A = torch.einsum("hj,jhd->hd", w, vv.abs())
        lg = vs[pg, :, j % page].double().log2().abs().clamp(max=150).amax()
        eps = (2 * S * (2.0 ** -19 + 2.0 ** -21 + 2.0 ** -22) + 2.0 ** -20 + 2.0 ** -21 + lg * 2.0 ** -22
               + (1.45 * S + lg) * 2.0 ** -24 + t / 16 * 2.0 ** -23 + 2.0 ** -19)
        # A weight times its scale is a sum of two f16, whose last step is 2^-24, where the largest of them stands at 2^7
        # or above (off by 2^-25 at most, 2^-32 of the largest), or, with one or two heads to a KV head, a whole number
        # where the largest stands at 2^29 or above: off by half, 2^-30 of the largest. That shows where the heavy rows'
        # integers are 0.
        vsc = vs[pg, :, j % page].double().T.repeat_interleave(H // kvh, 0)
        ints = v[pg, :, j % page].double().abs().sum(0).repeat_interleave(H // kvh, 0)
        small = 2.0 ** (-30 if H // kvh <= 2 else -32) * (w * vsc).amax(-1, keepdim=True) * ints
        ys.append(y)
        tols.append(small + 2 * A * eps + HALF_STEP[io] * y.abs() + (2.0 ** -25 if io == "f16" else 1e-30))
    return torch.stack(ys), torch.stack(tols)


# ---- attention -------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
def test_decode(lens, heads, io):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    page = [16, 32, 64, 256][(len(lens) + heads[0]) % 4]
    cache = make_q8(torch, lens, page, heads[1], seed=len(lens))
    q = (torch.randn(len(lens), heads[0], D, device="cuda") * 1.5).to(_types(torch)[io])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode_q8(q, *cache, status=status)
    want, tol = plain(torch, q, *cache, 0, 0, D ** -0.5, io)
    close(torch, y, want, tol)
    assert int(status) == 0 and bool((y[cache[-1] == 0] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 4), (100, 64), (64, 65), (1000, 1), (5000, 7), (130, 3000)])
@pytest.mark.parametrize("page", [16, 128])
def test_window_and_sinks_with_freed_pages(window, sinks, page):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [1500, 3, 150, 64, 1, 129]
    cache = make_q8(torch, lens, page, 2)
    table = cache[4]
    for b, t in enumerate(lens):   # a server frees the pages that no later query sees
        for i in range(table.shape[1]):
            lo, hi = i * page, min((i + 1) * page, t)
            if hi <= lo or (hi <= t - window and lo >= sinks):
                table[b, i] = -5 if i % 2 else 10 ** 6
    q = torch.randn(len(lens), 8, D, device="cuda") * 1.5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode_q8(q, *cache, window=window, sinks=sinks, status=status)
    want, tol = plain(torch, q, *cache, window, sinks, D ** -0.5, "f32")
    close(torch, y, want, tol)
    assert int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [30.0, 60.0])
@pytest.mark.parametrize("heavy", [False, True])
def test_scales_of_any_size(spread, heavy):
    """V rows 2^120 apart; heavy: the likeliest key's V is the smallest (as many models' first token)."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [300, 17, 1000]
    k, v, ks, vs, table, n = make_q8(torch, lens, 32, 2, seed=3, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(9)
    vs *= 2.0 ** ((torch.rand(vs.shape, generator=g, device="cuda") * 2 - 1) * spread)
    vs[:, 1, ::3] = torch.where(vs[:, 1, ::3].isnan(), vs[:, 1, ::3], 0.0)
    q = torch.randn(3, 8, D, device="cuda")
    if heavy:
        for b in range(3):
            k[table[b, 0], :, 0] = (q[b, ::4] * 30).clamp(-127, 127).to(torch.int8)
            ks[table[b, 0], :, 0] = 0.2
            vs[table[b, 0], :, 0] = 2.0 ** -spread
    y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
    want, tol = plain(torch, q, k, v, ks, vs, table, n, 0, 0, D ** -0.5, "f32")
    close(torch, y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [0.0, 1e-20, 1e5, 1e20])
@pytest.mark.parametrize("sign", [1, -1])
def test_queries_and_scales_of_any_size(size, sign):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    cache = make_q8(torch, [200, 65], 16, 2, seed=5)
    q = torch.randn(2, 4, D, device="cuda") * size
    scale = sign * D ** -0.5 / (size or 1.0)
    y = R.paged_attn_decode_q8(q, *cache, scale=scale)
    want, tol = plain(torch, q, *cache, 0, 0, torch.tensor(scale, dtype=torch.float32).double().item(), "f32")
    close(torch, y, want, tol)


@pytest.mark.gpu
def test_rows_that_are_not_finite_reach_only_who_sees_them():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, ks, vs, table, n = make_q8(torch, [100, 100], 16, 2)
    q = torch.randn(2, 4, D, device="cuda")
    clean = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
    for scales in (ks, vs):
        keep = scales.clone()
        scales[table[1, 3], 1, 5] = math.nan
        y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
        assert torch.equal(y[0], clean[0]) and torch.equal(y[1, :2], clean[1, :2]) and bool(y[1, 2:].isnan().all())
        y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n, window=30, sinks=4)   # out of its sight
        assert bool(torch.isfinite(y).all())
        scales.copy_(keep)


@pytest.mark.gpu
def test_strides_workspace_stream_and_replay():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [900, 33, 2500, 1]
    cache = make_q8(torch, lens, 16, 2, width=200)
    n = cache[-1]
    wide = torch.randn(4, 16 * D + 64, device="cuda")
    q = wide[:, :16 * D].unflatten(1, (16, D))
    out = torch.full((4, 16 * D + 8), 7.0, device="cuda")
    y = out[:, :16 * D].unflatten(1, (16, D))
    ws = torch.full((_lib.load().qd_paged_attn_decode_workspace_bytes(4, 16),), 255, dtype=torch.uint8, device="cuda")
    want = R.paged_attn_decode_q8(q.contiguous(), *cache)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    R.paged_attn_decode_q8(q, *cache, y=y, workspace=ws, stream=s)
    s.synchronize()
    assert torch.equal(y, want) and bool((out[:, 16 * D:] == 7.0).all())
    with pytest.raises(ValueError, match="overlaps"):
        R.paged_attn_decode_q8(q, *cache, y=q)
    spaces = [torch.empty_like(ws) for _ in range(2)]
    ys, graphs = [torch.zeros(4, 16, D, device="cuda") for _ in range(2)], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            R.paged_attn_decode_q8(q, *cache, y=ys[i], workspace=spaces[i], window=1000 * i)
        graphs.append(graph)
    for shorter in (lens, [1, 32, 1200, 0]):
        n.copy_(torch.tensor(shorter, dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want, tol = plain(torch, q, *cache, 1000 * i, 0, D ** -0.5, "f32")
            close(torch, ys[i], want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4, 2), (8, 2), (16, 2)], ids=lambda h: f"{h[0]}q{h[1]}kv")
def test_copies_that_do_not_come_end_in_nan_and_a_status(heads):
    """Block 0's first warp withholds its first copies: its waits end after a second."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    cache = make_q8(torch, [2000, 700, 40], 64, heads[1])
    q = torch.randn(3, heads[0], D, device="cuda")
    want = R.paged_attn_decode_q8(q, *cache)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.load().qd_paged_inject_stall()
    y = R.paged_attn_decode_q8(q, *cache, status=status)
    gone = y.isnan().any(-1)
    assert int(status) == _lib.QD_PAGED_TIMEOUT and torch.equal(gone, y.isnan().all(-1))
    # block 0: units of the first sequence's first KV head
    assert bool(gone[0, :heads[0] // heads[1]].all()) and int(gone.sum()) < gone.numel()
    assert torch.equal(y[~gone], want[~gone])
    status.zero_()
    assert torch.equal(R.paged_attn_decode_q8(q, *cache, status=status), want) and int(status) == 0


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_left_out_and_flagged():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, ks, vs, table, n = make_q8(torch, [100, 40], 16, 2)
    q = torch.randn(2, 4, D, device="cuda")
    good = table.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (k.shape[0], -1):
        table[0, 2] = bad          # positions 32..47 of sequence 0 are left out, as a window and sinks leave them out
        y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n, status=status)
        assert int(status) == _lib.QD_PAGED_BAD_PAGE
        want, tol = plain(torch, q, k, v, ks, vs, good, n, 100 - 48, 32, D ** -0.5, "f32")
        close(torch, y[:1], want[:1], tol[:1])
        status.zero_()
    table.copy_(good)
    n[0] = 10 ** 9                 # cut to the table
    y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_LENGTH
    status.zero_()
    n[0] = -3
    y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_LENGTH and bool((y[0] == 0).all())
    empty = [x[:0] for x in (k, v, ks, vs)]   # no pool at all
    status.zero_()
    y = R.paged_attn_decode_q8(q, *empty, table, n, status=status)
    assert int(status) & _lib.QD_PAGED_BAD_PAGE and bool((y == 0).all())


# ---- writing and reading back ------------------------------------------------------------------

def check_rows(torch, x, ints, scales, tol):
    """Rows x (64 bits, off by tol) against their 8-bit form."""
    top = x.abs().amax(-1)
    assert bool(((scales.double() * 127 - top).abs() <= tol.amax(-1) + 2.0 ** -22 * top).all())
    step = scales.double()[..., None]
    off = (x - ints.double() * step).abs()
    assert bool((off <= step * (0.5 + 127 * 2.0 ** -22) + 2 * tol + 2.0 ** -22 * x.abs()).all())
    assert int(ints.abs().max()) <= 127 and bool((ints.abs().amax(-1) == 127).all())


@pytest.mark.gpu
@pytest.mark.parametrize("io,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("new,totals", [([1], [9]), ([1, 1, 1], [5, 1, 700]), ([40, 0, 3, 129], [40, 7, 300, 129]),
                                        ([1] * 200, list(range(1, 201)))], ids=["one", "three", "ragged", "many"])
@pytest.mark.parametrize("heads", [(16, 8), (5, 1), (0, 2)], ids=lambda h: f"{h[0]}q{h[1]}kv")
def test_append(io, out, new, totals, heads):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    T = _types(torch)
    H, kvh = heads
    k, v, ks, vs, table, n = make_q8(torch, totals, 16, kvh, fill=False)
    rows, pad = sum(new), 2
    qkv = torch.randn(rows + pad, (H + 2 * kvh) * D + 24, device="cuda").to(T[io])[:, :(H + 2 * kvh) * D]
    qn, kn = torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda") + 0.5
    angle = torch.rand(max(totals), 64, device="cuda") * 6.28
    cos, sin = angle.cos(), angle.sin()
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    q_out = torch.full((rows + pad, H * D), 3.0, device="cuda").to(T[out])
    before = [x.clone() for x in (k, v, ks, vs)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    R.paged_append_q8(qkv, k, v, ks, vs, table, n, cos, sin, H, q_norm=qn, k_norm=kn, q_starts=starts, q_out=q_out,
                      status=status)
    assert int(status) == 0 and bool((q_out[rows:] == 3).all())
    # q is paged_append's to the bit
    k16, v16 = (torch.zeros(k.shape, dtype=torch.float16, device="cuda") for _ in "kv")
    same = torch.full_like(q_out, 3.0)
    R.paged_append(qkv, k16, v16, table, n, cos, sin, H, q_norm=qn, k_norm=kn, q_starts=starts, q_out=same)
    assert torch.equal(q_out, same)
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(t - m, t) for m, t in zip(new, totals)]).cuda()
    pg = table[seq].long().gather(1, (pos // 16)[:, None])[:, 0]
    x = qkv[:rows].double().unflatten(1, (-1, D))
    h = x[:, H:H + kvh]
    h = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * kn.double()
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = h[..., :64], h[..., 64:]
    tol = 16 * 2.0 ** -24 * torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    check_rows(torch, torch.cat([a * c - b * s, b * c + a * s], -1), k[pg, :, pos % 16], ks[pg, :, pos % 16], tol)
    val = x[:, H + kvh:]
    check_rows(torch, val, v[pg, :, pos % 16], vs[pg, :, pos % 16], torch.zeros_like(val))
    untouched = torch.ones(k.shape[0], k.shape[2], dtype=torch.bool, device="cuda")
    untouched[pg, pos % 16] = False
    for now, was in zip((k, v, ks, vs), before):
        assert torch.equal(now.transpose(1, 2)[untouched], was.transpose(1, 2)[untouched])


@pytest.mark.gpu
def test_rows_without_a_scale_of_their_own():
    """Zeros, tiny, huge and non-finite rows, and one whose elements are halves between two integers."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    rows = torch.zeros(9, D, device="cuda")
    rows[1] = torch.randn(D, device="cuda") * 1e-38            # below 2^-100
    rows[2] = torch.randn(D, device="cuda") * 1e-25
    rows[3] = torch.randn(D, device="cuda") * 1e37
    rows[4] = torch.randn(D, device="cuda")
    rows[5] = rows[4].clone()
    rows[5, 77] = math.inf
    rows[6] = rows[4].clone()
    rows[6, 3] = math.nan
    rows[7] = torch.arange(D, device="cuda") - 63.5            # scale 1 / 2: whole numbers times 2, and
    rows[8, :2] = torch.tensor([-127.0, 2.5], device="cuda")   # a tie: to the even one
    rows[7, 127] = 63.5
    k8, v8 = (torch.full((1, 1, 16, D), 9, dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.full((1, 1, 16), 7.0, device="cuda") for _ in "kv")
    qkv = torch.cat([torch.zeros_like(rows), rows], 1)
    n = torch.tensor([9], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    R.paged_append_q8(qkv, k8, v8, ks, vs, table, n, None, None, 0, q_starts=starts)
    assert bool((k8[0, 0, :9] == 0).all()) and bool((ks[0, 0, :9] == 0).all())
    assert bool((v8[0, 0, 9:] == 9).all()) and bool((vs[0, 0, 9:] == 7).all())
    s = vs[0, 0, :9]
    assert s[0] == 0 and s[1] == 0 and bool((v8[0, 0, :2] == 0).all())
    assert bool(s[5:7].isnan().all())
    check_rows(torch, rows[2:5].double(), v8[0, 0, 2:5], s[2:5], torch.zeros(3, D, device="cuda", dtype=torch.float64))
    assert s[7] == 0.5 and torch.equal(v8[0, 0, 7].float(), rows[7] * 2)
    assert s[8] == 1 and v8[0, 0, 8, 0] == -127 and v8[0, 0, 8, 1] == 2
    out = [torch.full((1, 1, 16, D), 5.0, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    R.paged_read_q8(k8, v8, ks, vs, table, n, *out, table)
    assert bool((out[1][0, 0, :2] == 0).all()) and bool(out[1][0, 0, 5:7].isnan().all())
    assert torch.equal(out[1][0, 0, 7], rows[7].bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("lens,first", [([1], None), ([31], [15]), ([0, 700, 16, 17, 3], [0, 3, 16, 16, 2]),
                                        ([5] * 300, None), ([9000, 40], [-5, 50])], ids=["1", "31", "ragged", "many", "long"])
@pytest.mark.parametrize("pages", [(16, 16), (64, 16), (16, 256)], ids=str)
def test_read(lens, first, cache, pages):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, ks, vs, table, n = make_q8(torch, lens, pages[0], 3, seed=7)
    width = max(-(-t // pages[1]) for t in lens) + 1
    out_table = torch.randperm(len(lens) * width, device="cuda").to(torch.int32).view(len(lens), width)
    T = _types(torch)[cache]
    out = [torch.full((len(lens) * width, 3, pages[1], D), 5.0, device="cuda", dtype=T) for _ in "kv"]
    want = [x.clone() for x in out]
    for b, t in enumerate(lens):
        j = torch.arange(min(max(first[b], 0), t) if first else 0, t, device="cuda")
        src, dst = table[b].long()[j // pages[0]], out_table[b].long()[j // pages[1]]
        for x, s, y in ((k, ks, want[0]), (v, vs, want[1])):
            y[dst, :, j % pages[1]] = (x[src, :, j % pages[0]].float() * s[src, :, j % pages[0]][..., None]).to(T)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    f = torch.tensor(first, dtype=torch.int32, device="cuda") if first else None
    got = R.paged_read_q8(k, v, ks, vs, table, n, *out, out_table, first=f, status=status)
    assert int(status) == 0 and got[0] is not None
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.gpu
def test_reading_flags_what_has_no_place():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, ks, vs, table, n = make_q8(torch, [60, 20], 16, 2)
    out = [torch.zeros(8, 2, 16, D, device="cuda", dtype=torch.float16) for _ in "kv"]
    out_table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def read(tab, to):
        status.zero_()
        for x in out:
            x.fill_(5.0)
        R.paged_read_q8(k, v, ks, vs, tab, n, *out, to, status=status)
        return int(status)

    assert read(table, out_table) == 0
    whole = [x.clone() for x in out]
    for side in (0, 1):
        tabs = [table.clone(), out_table.clone()]
        tabs[side][0, 1] = 8 + k.shape[0]
        assert read(*tabs) == _lib.QD_PAGED_BAD_PAGE
        for x, w in zip(out, whole):
            assert bool((x[1] == 5).all()) and torch.equal(x[2:], w[2:]) and torch.equal(x[0], w[0])
    assert read(table, out_table[:, :2].contiguous()) == _lib.QD_PAGED_BAD_LENGTH    # cut to the target's table
    assert torch.equal(out[0][:2], whole[0][:2])
    n[1] = -1
    assert read(table, out_table) == _lib.QD_PAGED_BAD_LENGTH and bool((out[0][4:] == 5).all())


# ---- together -----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 24])
def test_prompts_then_decoding_steps_over_an_8_bit_cache(window):
    """Chunked prompts: appended in 8 bits, read back for the prompt's attention (the pages of a chunk are
    scratch); then single tokens."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    from test_paged import plain_attention
    torch.manual_seed(5)
    H, kvh, page, sinks = 8, 2, 16, 4
    k, v = (torch.zeros(40, kvh, page, D, device="cuda", dtype=torch.int8) for _ in "kv")
    ks, vs = (torch.full((40, kvh, page), math.nan, device="cuda") for _ in "kv")
    table = torch.randperm(40, device="cuda")[:36].to(torch.int32).view(3, 12)
    a = torch.outer(torch.arange(192, device="cuda").double(), 1e6 ** (-torch.arange(64, device="cuda").double() / 64))
    cos, sin = a.cos().float(), a.sin().float()
    held = torch.zeros(3, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    scratch = [torch.full((18, kvh, 32, D), math.nan, device="cuda", dtype=torch.float16) for _ in "kv"]
    scratch_table = torch.arange(18, dtype=torch.int32, device="cuda").view(3, 6)
    for new in ([70, 3, 33], [41, 1, 0], [1, 1, 1], [1, 1, 1]):
        held += torch.tensor(new, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32, device="cuda")
        qkv = torch.randn(sum(new), (H + 2 * kvh) * D, device="cuda")
        q = R.paged_append_q8(qkv, k, v, ks, vs, table, held, cos, sin, H, q_starts=starts, status=status).view(-1, H, D)
        if max(new) > 1:
            R.paged_read_q8(k, v, ks, vs, table, held, *scratch, scratch_table, status=status)
            y = R.paged_attn_prompt(q, *scratch, scratch_table, held, starts, window=window, sinks=sinks, status=status)
            want, tol = plain_attention(torch, q, *scratch, scratch_table, held, new, window, sinks, D ** -0.5, "f32", "f16")
        else:
            y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, held, window=window, sinks=sinks, status=status)
            want, tol = plain(torch, q, k, v, ks, vs, table, held, window, sinks, D ** -0.5, "f32")
        close(torch, y, want, tol)
    assert int(status) == 0


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pools of 4.6 GB (scales 1.2 GB among them) whose used pages lie at both ends."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    pages, kvh, page, H = 70000, 8, 64, 16
    k, v = (torch.empty(pages, kvh, page, D, dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.empty(pages, kvh, page, device="cuda") for _ in "kv")
    small = make_q8(torch, [300, 131], page, kvh)
    used = torch.unique(small[4][small[4] >= 0]).long()
    far = torch.where(used % 2 == 0, pages - 1 - used, used)
    for big, x in zip((k, v, ks, vs), small):
        big[far] = x[used]
    table, n = small[4].clone(), small[5]
    for a, b in zip(used.tolist(), far.tolist()):
        table[small[4] == a] = b
    qkv = torch.randn(2, (H + 2 * kvh) * D, device="cuda")
    want = R.paged_append_q8(qkv, *small, None, None, H).view(2, H, D)
    got = R.paged_append_q8(qkv, k, v, ks, vs, table, n, None, None, H).view(2, H, D)
    assert torch.equal(got, want)
    for big, x in zip((k, v, ks, vs), small):
        assert torch.equal(big[far].nan_to_num(), x[used].nan_to_num())
    assert torch.equal(R.paged_attn_decode_q8(got, k, v, ks, vs, table, n), R.paged_attn_decode_q8(want, *small))
    outs = [[torch.zeros(12, kvh, page, D, dtype=torch.float16, device="cuda") for _ in "kv"] for _ in range(2)]
    to = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    R.paged_read_q8(k, v, ks, vs, table, n, *outs[0], to)
    R.paged_read_q8(*small, *outs[1], to)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1.0, 1e-3, 200.0])
def test_integers_are_the_quotients_rounded(io, size):
    """n = 127 x / max|x| rounded, halves to even: every integer of rows in which many elements are halves (of the largest,
    and between any two integers of rows whose largest is 127 times a power of two). In 16 bits no quotient comes nearer
    to a half than 2^-19 of itself without being one, and a quotient is off by 2^-24 of itself; in f32 only the
    halves, and what lies 2^-16 of a step from one, are compared."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    rows, kvh = 300, 4
    T = _types(torch)[io]
    g = torch.Generator(device="cuda").manual_seed(11)
    x = (torch.randn(rows, 2 * kvh, D, generator=g, device="cuda") * size).to(T)
    top = x.abs().amax(-1, keepdim=True)
    x[:, :, 5:40:3] = top * 0.5 * torch.randn(rows, 2 * kvh, 12, generator=g, device="cuda").sign().to(T)
    odd = 2 * torch.randint(-127, 127, (rows // 2, 2 * kvh, D), generator=g, device="cuda") + 1
    x[::2] = (odd * 0.5 if size == 1.0 else odd * 0.0625).to(T)   # at most 126.5 or an eighth of it, exact in 8 bits and more
    x[::2, :, 9] = 127.0 if size == 1.0 else -127.0 / 8
    k8, v8, ks, vs, table, n = make_q8(torch, [rows], 64, kvh, fill=False)
    starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    R.paged_append_q8(x.flatten(1), k8, v8, ks, vs, table, n, None, None, 0, q_starts=starts)
    at = torch.arange(rows, device="cuda")
    pg = table[0].long()[at // 64]
    ints = torch.cat([k8[pg, :, at % 64], v8[pg, :, at % 64]], 1)
    scales = torch.cat([ks[pg, :, at % 64], vs[pg, :, at % 64]], 1)
    most = x.double().abs().amax(-1)
    assert bool(((scales.double() * 127 - most).abs() <= 2.0 ** -24 * 1.001 * most).all())   # half a step
    q = x.double() * 127 / most[..., None]
    off = ((q - q.floor()) - 0.5).abs()
    assert int((off == 0).sum()) > rows * kvh * 32
    sure = (off == 0) | (off > 2.0 ** -16) if io == "f32" else torch.ones_like(off, dtype=torch.bool)
    assert torch.equal(ints[sure].double(), q.round()[sure])


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-125, -118, -105, -97, -90, 0, 100])
@pytest.mark.parametrize("heads", [4, 8, 16], ids=lambda h: f"{h}q2kv")
def test_v_scales_down_to_the_smallest(exponent, heads):
    """Every V scale within a factor of 2 of 2^exponent: results go down to 2^-126 and are not flushed. (The tolerance's
    term for the smallest numbers makes place for 4 of f32's last ones.)"""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [300, 1, 5000, 17]
    k, v, ks, vs, table, n = make_q8(torch, lens, 32, 2, seed=21, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(4)
    vs *= 0.0
    vs += torch.ldexp(1 + torch.rand(vs.shape, generator=g, device="cuda"), torch.tensor(exponent, device="cuda"))
    q = torch.randn(len(lens), heads, D, device="cuda")
    y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
    want, tol = plain(torch, q, k, v, ks, vs, table, n, 0, 0, D ** -0.5, "f32")
    close(torch, y, want, tol - 1e-30 + 2.0 ** -147)
    assert bool((y != 0).any(-1).all())


KERNELS = pytest.mark.parametrize("heads", [4, 8, 16], ids=lambda h: f"{h}q2kv")   # one for each kernel behind the call


@pytest.mark.gpu
@KERNELS
@pytest.mark.parametrize("spread", [30.0, 60.0])
@pytest.mark.parametrize("heavy", [False, True])
def test_scales_of_any_size_in_every_kernel(heads, spread, heavy):
    """V rows 2^120 apart, some of them zeros; heavy: the likeliest key's V is the smallest, for every head."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [300, 17, 1000]
    k, v, ks, vs, table, n = make_q8(torch, lens, 32, 2, seed=3, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(9)
    vs *= 2.0 ** ((torch.rand(vs.shape, generator=g, device="cuda") * 2 - 1) * spread)
    vs[:, 1, ::3] = torch.where(vs[:, 1, ::3].isnan(), vs[:, 1, ::3], 0.0)
    q = torch.randn(3, heads, D, device="cuda")
    if heavy:
        q = q[:, ::heads // 2].repeat_interleave(heads // 2, 1) + 0.1 * q
        for b in range(3):
            k[table[b, 0], :, 0] = (q[b, ::heads // 2] * 30).clamp(-127, 127).to(torch.int8)
            ks[table[b, 0], :, 0] = 0.2
            vs[table[b, 0], :, 0] = 2.0 ** -spread
    y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
    want, tol = plain(torch, q, k, v, ks, vs, table, n, 0, 0, D ** -0.5, "f32")
    close(torch, y, want, tol)


@pytest.mark.gpu
@KERNELS
@pytest.mark.parametrize("size", [0.0, 1e-20, 1e5, 1e20])
@pytest.mark.parametrize("sign", [1, -1])
def test_queries_of_any_size_in_every_kernel(heads, size, sign):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    cache = make_q8(torch, [200, 65], 16, 2, seed=5)
    q = torch.randn(2, heads, D, device="cuda") * size
    scale = sign * D ** -0.5 / (size or 1.0)
    y = R.paged_attn_decode_q8(q, *cache, scale=scale)
    want, tol = plain(torch, q, *cache, 0, 0, torch.tensor(scale, dtype=torch.float32).double().item(), "f32")
    close(torch, y, want, tol)


@pytest.mark.gpu
@KERNELS
def test_rows_that_are_not_finite_in_every_kernel(heads):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, ks, vs, table, n = make_q8(torch, [100, 100], 16, 2)
    q = torch.randn(2, heads, D, device="cuda")
    G = heads // 2
    clean = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
    for scales in (ks, vs):
        keep = scales.clone()
        for bad in (math.nan, math.inf):
            scales[table[1, 3], 1, 5] = bad
            y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
            assert torch.equal(y[0], clean[0]) and torch.equal(y[1, :G], clean[1, :G])
            if bad != bad or scales is vs:   # (an infinite key may have a weight of 0)
                assert not bool(torch.isfinite(y[1, G:]).any())
            y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n, window=30, sinks=4)   # out of its sight
            assert bool(torch.isfinite(y).all())
        scales.copy_(keep)
    q[0, 1, 3] = math.nan   # a query of its own
    y = R.paged_attn_decode_q8(q, k, v, ks, vs, table, n)
    assert bool(y[0, 1].isnan().all()) and bool(torch.isfinite(y[0, 0]).all()) and torch.equal(y[1], clean[1])


@pytest.mark.gpu
@KERNELS
@pytest.mark.parametrize("window,sinks", [(1, 0), (17, 4), (64, 65), (130, 3000)])
def test_window_and_sinks_in_every_kernel(heads, window, sinks):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [1500, 3, 150, 64, 1, 129]
    cache = make_q8(torch, lens, 16, 2)
    q = torch.randn(len(lens), heads, D, device="cuda") * 1.5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode_q8(q, *cache, window=window, sinks=sinks, status=status)
    want, tol = plain(torch, q, *cache, window, sinks, D ** -0.5, "f32")
    close(torch, y, want, tol)
    assert int(status) == 0
