"""The paged key-value cache operators (qd_paged_append, qd_paged_attn_decode,
qd_paged_attn_prompt): refusals on the host (no GPU), and the CUDA path against plain
64-bit evaluations at the sizes, masks and layouts where it can go wrong.

Tolerances count roundings, relative to A = sum of |weight| |value| of an output:
 - a score is a sum of 128 products: its error is at most S e_s, S = scale * sum |q| |k|,
   e_s = 2^-19 for the f32 accumulation (8 steps of 16 products, one truncation of 2^-23
   each, two operand parts) plus the operands' split (2^-21 for f32 as two f16, 2^-16 as two
   bf16, 0 where q is 16-bit);
 - a weight exp(s - m) is then off by 2 S e_s (score and maximum), plus 2^-20 for the
   exponential and its rounded argument, plus its own rounding where it feeds a product in 16
   bits (half a step: 2^-11, 2^-8) or as a sum of two parts (2^-21, 2^-16);
 - sums over n keys in f32, in steps of 16 keys or fewer joins: n / 16 * 2^-23 + 2^-19;
 - the output's own rounding, half a step of its type."""
import ctypes as C
import math
import random
import subprocess
import sys
import textwrap
import threading

import pytest

from kernel_optimization_webgpu_b200 import _lib

D = 128
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# ---- refusals (no GPU) -----------------------------------------------------------------

def _kv(**kw):
    d = dict(k=4096, v=8192, dtype=_lib.QD_KV_F16, num_pages=4, page_size=16, kv_heads=2, head_dim=128, batch=2,
             block_table=4096, table_width=3, table_stride=3, seq_lens=4096, status=None)
    d.update(kw)
    return _lib.QdPagedKv(*(d[n] for n, _ in _lib.QdPagedKv._fields_))


BAD_CACHES = [dict(dtype=_lib.QD_KV_F32), dict(dtype=7), dict(page_size=24), dict(page_size=8), dict(page_size=512),
              dict(head_dim=64), dict(kv_heads=0), dict(batch=-1), dict(batch=4097), dict(num_pages=-1),
              dict(table_stride=2), dict(table_width=-1, table_stride=0), dict(block_table=None), dict(seq_lens=None),
              dict(k=None), dict(v=8200), dict(table_width=1 << 27, table_stride=1 << 27)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_a_bad_cache_is_refused_by_every_entry(bad):
    L = _lib.load()
    kv = _kv(**bad)
    assert L.qd_paged_append(kv, 4096, 1, 768, 2, None, 2, None, None, 1e-6, None, None, 0, 0, 4096, 1, 256,
                             None) == _lib.QD_E_INVALID
    assert L.qd_paged_attn_decode(kv, 4096, 1, 256, 2, 0, 0, 0.0, 4096, 256, 4096, None) == _lib.QD_E_INVALID
    assert L.qd_paged_attn_prompt(kv, 4096, 1, 256, 2, 4096, 2, 0, 0, 0.0, 4096, 256, 4096, None) == _lib.QD_E_INVALID
    assert L.qd_last_error(None).startswith(b"paged cache")


def test_attention_arguments_are_refused():
    L = _lib.load()
    ok = dict(q=4096, dtype=1, stride=256, heads=2, window=0, sinks=0, scale=0.0, y=8192, y_stride=256, ws=4096)
    bads = [dict(q=None), dict(y=None), dict(ws=None), dict(q=4104), dict(dtype=2), dict(dtype=9), dict(stride=248),
            dict(stride=260), dict(y_stride=128), dict(heads=3), dict(heads=0), dict(heads=130), dict(window=-1),
            dict(sinks=-1), dict(scale=math.inf), dict(scale=math.nan)]
    for bad in bads:
        c = {**ok, **bad}
        if bad.get("heads") == 130:
            c.update(stride=130 * 128, y_stride=130 * 128)
        rc = L.qd_paged_attn_decode(_kv(), c["q"], c["dtype"], c["stride"], c["heads"], c["window"], c["sinks"],
                                    c["scale"], c["y"], c["y_stride"], c["ws"], None)
        assert rc == _lib.QD_E_INVALID, bad
        rc = L.qd_paged_attn_prompt(_kv(), c["q"], c["dtype"], c["stride"], 5, 4096, c["heads"], c["window"], c["sinks"],
                                    c["scale"], c["y"], c["y_stride"], c["ws"], None)
        assert rc == _lib.QD_E_INVALID, bad
    assert L.qd_paged_attn_decode(None, 4096, 1, 256, 2, 0, 0, 0.0, 4096, 256, 4096, None) == _lib.QD_E_INVALID
    assert L.qd_paged_attn_prompt(_kv(), 4096, 1, 256, 5, None, 2, 0, 0, 0.0, 4096, 256, 4096,
                                  None) == _lib.QD_E_INVALID
    assert L.qd_paged_attn_prompt(_kv(), 4096, 1, 256, -1, 4096, 2, 0, 0, 0.0, 4096, 256, 4096,
                                  None) == _lib.QD_E_INVALID
    # nothing to do is not an error, and touches nothing
    assert L.qd_paged_attn_prompt(_kv(), None, 1, 256, 0, None, 2, 0, 0, 0.0, None, 256, None, None) == _lib.QD_OK
    assert L.qd_paged_attn_decode(_kv(batch=0), None, 1, 256, 2, 0, 0, 0.0, None, 256, None, None) == _lib.QD_OK


def test_append_arguments_are_refused():
    L = _lib.load()
    ok = dict(qkv=4096, dtype=1, stride=768, rows=2, starts=None, heads=2, qn=None, kn=None, eps=1e-6, cos=4096, sin=4096,
              rope_len=640, rope_stride=64, out=4096, out_dtype=1, out_stride=256)
    bads = [dict(qkv=None), dict(out=None), dict(qkv=4100), dict(out=4104), dict(dtype=3), dict(out_dtype=-1),
            dict(stride=760), dict(stride=770), dict(rows=-1), dict(rows=3), dict(heads=-1), dict(eps=-1.0),
            dict(eps=math.nan), dict(sin=None), dict(cos=None), dict(rope_stride=2), dict(rope_stride=-64),
            dict(rope_len=-1), dict(out_stride=128), dict(qn=4100), dict(kn=4100), dict(cos=4100)]
    for bad in bads:
        c = {**ok, **bad}
        rc = L.qd_paged_append(_kv(), c["qkv"], c["dtype"], c["stride"], c["rows"], c["starts"], c["heads"], c["qn"],
                               c["kn"], c["eps"], c["cos"], c["sin"], c["rope_len"], c["rope_stride"], c["out"],
                               c["out_dtype"], c["out_stride"], None)
        assert rc == _lib.QD_E_INVALID, bad
    assert L.qd_paged_append(_kv(), None, 1, 768, 0, 4096, 2, None, None, 1e-6, None, None, 0, 0, None, 1, 256,
                             None) == _lib.QD_OK


def test_python_wrappers_refuse_before_they_enqueue():
    torch = pytest.importorskip("torch")
    from kernel_optimization_webgpu_b200 import runtime as R
    k = torch.zeros(4, 2, 16, D, dtype=torch.float16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 2, D)
    for args in ((q, k, k[:3], table, lens), (q, k, k.bfloat16(), table, lens), (q, k.transpose(1, 2), k, table, lens),
                 (q, k, k, table.long(), lens), (q, k, k, table, lens.long()), (q, k, k, table, lens[:1]),
                 (q[:1], k, k, table, lens), (q[..., :64], k, k, table, lens), (q.transpose(0, 1), k, k, table, lens),
                 (q.double(), k, k, table, lens), (q, k, k, table, lens)):   # the last: not CUDA tensors
        with pytest.raises(ValueError):
            R.paged_attn_decode(*args)
    with pytest.raises(ValueError):
        R.paged_append(torch.zeros(2, 700), k, k, table, lens, None, None, 2)


BASE = 1 << 40   # (addresses that nothing is read from)


def _refuses(call, *args):
    """Whether a call over sequences without a row to work on is refused, and with which words."""
    rc = call(*args)
    assert rc in (_lib.QD_OK, _lib.QD_E_INVALID)
    return _lib.load().qd_last_error(None).decode() if rc else ""


@pytest.mark.parametrize("dy,stride,y_stride,batch,over", [
    (0, 256, 256, 2, "q"), (512, 256, 256, 2, "q"), (1024, 256, 256, 2, ""), (-512, 256, 256, 2, "q"),
    (-1024, 256, 256, 2, ""), (512, 512, 512, 2, ""), (496, 512, 512, 2, "q"), (528, 512, 512, 2, "q"),
    (512, 520, 520, 2, ""), (1552, 520, 520, 2, ""), (512, 512, 256, 2, "q"), (512, 512, 256, 1, ""),
    (0, 512, 256, 1, "q"), (BASE, 256, 256, 2, "the pools"), (BASE - 16, 256, 256, 2, "the pools"),
    (BASE + 32768 - 16, 256, 256, 2, "the pools"), (BASE + 32768, 256, 256, 2, ""), (2 * BASE, 256, 256, 2, "the pools")])
def test_attention_outputs_over_their_inputs_are_refused(dy, stride, y_stride, batch, over):
    """q at BASE, 512-byte rows; pools of 32768 bytes at 2 and 3 BASE. A NULL workspace ends what is not refused."""
    L = _lib.load()
    kv = _kv(k=2 * BASE, v=3 * BASE, batch=batch, block_table=64, seq_lens=64)
    args = (kv, BASE, _lib.QD_KV_F16, stride, 2, 0, 0, 0.0, BASE + dy, y_stride, None, None)
    assert _refuses(L.qd_paged_attn_decode, *args) == (
        f"paged attention: y overlaps {over}" if over else "qd_paged_attn_decode: NULL workspace")
    # of a ragged batch the rows behind the first may be padding without memory
    if -512 < dy < 512 or over != "q":
        args = (kv, BASE, _lib.QD_KV_F16, stride, batch, 64, 2, 0, 0, 0.0, BASE + dy, y_stride, None, None)
        assert _refuses(L.qd_paged_attn_prompt, *args) == (
            f"paged attention: y overlaps {over}" if over else "qd_paged_attn_prompt: NULL workspace")


@pytest.mark.parametrize("out,dtype,stride,over", [
    (BASE, 1, 768, ""), (BASE, 1, 776, "q_out overlaps qkv"), (BASE, 0, 768, "q_out overlaps qkv"),
    (BASE + 256, 1, 768, "q_out overlaps qkv"), (BASE + 768 * 4, 1, 768, "q_out overlaps qkv"),
    (BASE + 2 * 768 * 4, 1, 768, ""), (2 * BASE, 1, 768, "q_out overlaps the pools"),
    (3 * BASE + 32000, 0, 768, "q_out overlaps the pools")])
def test_append_outputs_over_their_inputs_are_refused(out, dtype, stride, over):
    """qkv at BASE, two rows of 768 f32. A cache that nothing is written to: eps ends what is not refused."""
    kv = _kv(k=2 * BASE, v=3 * BASE, block_table=64, seq_lens=64)
    L = _lib.load()

    def call(eps):
        return _refuses(L.qd_paged_append, kv, BASE, _lib.QD_KV_F32, 768, 2, None, 2, None, None, eps, None, None, 0, 0, out,
                        dtype, stride, None)

    assert "eps" in call(-1.0)
    if over:
        assert over in call(1e-6)
    else:   # the same layout over a cache of no sequences is no error
        kv.batch = 0
        assert _refuses(L.qd_paged_append, kv, BASE, _lib.QD_KV_F32, 768, 2, 64, 2, None, None, 1e-6, None, None, 0, 0, out,
                        dtype, stride, None) == ""


@pytest.mark.gpu
def test_outputs_beside_their_inputs_in_one_buffer():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [50, 3], 16, 2, "f16")
    both = torch.randn(2, 2, 4, D, device="cuda")
    q, y = both[:, 0], both[:, 1]
    want = R.paged_attn_decode(q.clone(), k, v, table, n)
    assert torch.equal(R.paged_attn_decode(q, k, v, table, n, y=y), want) and torch.equal(y, want)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    three = torch.randn(3, 4, D, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        R.paged_attn_decode(q, k, v, table, n, y=q)
    with pytest.raises(ValueError, match="overlaps"):
        R.paged_attn_prompt(three[:2], k, v, table, n, starts, y=three[1:])
    pool = k.view(torch.float32).reshape(-1)[:2 * 4 * D].view(2, 4, D)
    with pytest.raises(_lib.QdError, match="pools"):
        R.paged_attn_prompt(q, k, v, table, n, starts, y=pool)
    qkv = torch.randn(1, 8 * D, device="cuda")      # one row: its stride says nothing
    x = qkv.clone()
    R.paged_append(qkv, k, v, table[:1], n[:1], None, None, 4, q_out=qkv[:, :4 * D])
    assert torch.equal(qkv, x)
    with pytest.raises(ValueError, match="overlaps"):
        R.paged_append(qkv, k, v, table[:1], n[:1], None, None, 4, q_out=qkv[:, D:5 * D])


# ---- the plain 64-bit forms -------------------------------------------------------------

def _cuda():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _types(torch):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make_cache(torch, totals, page, kv_heads, cache, seed=0, slack=0, fill=None, width=None):
    """Pools of random rows, every page owned by one sequence or by none; a shuffled table.
    fill: what every row that no sequence holds contains (NaN, for instance)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = [-(-n // page) for n in totals]
    pages = sum(per) + 2 + slack
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = width or max(per + [1])
    table = torch.full((len(totals), width), -1, dtype=torch.int32)
    T = _types(torch)[cache]
    k, v = (torch.randn(pages, kv_heads, page, D, generator=g, device="cuda").to(T) for _ in "kv")
    if fill is not None:
        keep_k, keep_v = k.clone(), v.clone()
        k.fill_(fill), v.fill_(fill)
    at = 0
    for b, n in enumerate(per):
        for i in range(n):
            pg = order[at]
            at += 1
            table[b, i] = pg
            if fill is not None:
                m = min(page, totals[b] - i * page)
                k[pg, :, :m], v[pg, :, :m] = keep_k[pg, :, :m], keep_v[pg, :, :m]
    return k, v, table.cuda(), torch.tensor(totals, dtype=torch.int32, device="cuda")


def plain_attention(torch, q, k, v, table, lens, new, window, sinks, scale, io, cache):
    """(y, tolerance) in 64 bits; new[b]: sequence b's new tokens (rows in order)."""
    page, kvh = k.shape[2], k.shape[1]
    H = q.shape[1]
    ys, tols, first = [], [], 0
    split = 0.0 if io != "f32" else (2.0 ** -21 if cache == "f16" else 2.0 ** -16)
    weight = HALF_STEP[cache] if io != "f32" else split
    for b, n in enumerate(new):
        t = int(lens[b])
        qs = q[first:first + n].double()
        first += n
        j = torch.arange(max(t, 1), device="cuda")[:max(t, 0)]
        pg = table[b].long()[j // page]
        p = torch.arange(t - n, t, device="cuda")[:, None]
        seen = (j[None] <= p) & ((window == 0) | (j[None] > p - window) | (j[None] < sinks))
        seen_any = seen.any(0)
        pg = torch.where(seen_any, pg, torch.zeros_like(pg)) if t > 0 else pg
        kk = torch.where(seen_any[:, None, None], k[pg, :, j % page].double(), 0.0).repeat_interleave(H // kvh, 1)
        vv = torch.where(seen_any[:, None, None], v[pg, :, j % page].double(), 0.0).repeat_interleave(H // kvh, 1)
        s = torch.einsum("nhd,jhd->nhj", qs, kk) * scale
        size = torch.where(seen[:, None], torch.einsum("nhd,jhd->nhj", qs.abs(), kk.abs()) * abs(scale), 0.0)
        s = s.masked_fill(~seen[:, None], -math.inf)
        w = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300)) if t > 0 else s
        w = torch.where(seen[:, None], w, 0.0)
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
        y = torch.einsum("nhj,jhd->nhd", w, vv)
        A = torch.einsum("nhj,jhd->nhd", w, vv.abs())
        S = size.amax(-1)[..., None] if t > 0 else torch.zeros_like(y[..., :1])
        eps = 2 * S * (2.0 ** -19 + split) + 2.0 ** -20 + weight + max(t, 0) / 16 * 2.0 ** -23 + 2.0 ** -19
        ys.append(y)
        tols.append(2 * A * eps + HALF_STEP[io] * y.abs() + (2.0 ** -25 if io == "f16" else 1e-30))
    return torch.cat(ys), torch.cat(tols)


def close(torch, got, want, tol):
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).nan_to_num(math.inf).max()):.3g} tolerances"


# ---- attention of one new token ------------------------------------------------------------

LENS = [[1], [31], [64, 65, 63], [0, 1, 0, 17, 0], [2049, 5, 700, 129], [1] * 70, [4000]]
HEADS = [(16, 8), (8, 1), (4, 4), (10, 2), (12, 4), (18, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
def test_decode_attention(lens, heads, io, cache):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    page = [16, 32, 64, 256][(len(lens) + heads[0]) % 4]
    # every row that is nobody's holds NaN: recycled and unwritten pages reach no result
    k, v, table, n = make_cache(torch, lens, page, heads[1], cache, seed=len(lens), fill=math.nan)
    q = (torch.randn(len(lens), heads[0], D, device="cuda") * 1.5).to(_types(torch)[io])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode(q, k, v, table, n, status=status)
    want, tol = plain_attention(torch, q, k, v, table, n, [1] * len(lens), 0, 0, D ** -0.5, io, cache)
    close(torch, y, want, tol)
    assert int(status) == 0
    assert bool((y[n == 0] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 4), (100, 64), (64, 65), (1000, 1), (5000, 7), (130, 3000)])
@pytest.mark.parametrize("page", [16, 128])
def test_decode_window_and_sinks_with_freed_pages(window, sinks, page):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [1500, 3, 150, 64, 1]
    k, v, table, n = make_cache(torch, lens, page, 2, "f16", fill=math.nan)
    for b, t in enumerate(lens):   # a server frees the pages that no later query sees
        for i in range(table.shape[1]):
            lo, hi = i * page, min((i + 1) * page, t)
            if hi <= lo or (hi <= t - window and lo >= sinks):
                table[b, i] = -5 if i % 2 else 10 ** 6
    q = torch.randn(len(lens), 8, D, device="cuda") * 1.5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode(q, k, v, table, n, window=window, sinks=sinks, status=status)
    want, tol = plain_attention(torch, q, k, v, table, n, [1] * 5, window, sinks, D ** -0.5, "f32", "f16")
    close(torch, y, want, tol)
    assert int(status) == 0


@pytest.mark.gpu
def test_decode_strides_scale_workspace_and_stream():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [300, 7, 90]
    k, v, table, n = make_cache(torch, lens, 32, 4, "f16", width=40)
    wide = torch.randn(3, 8 * D + 64, device="cuda")
    q = wide[:, :8 * D].unflatten(1, (8, D))
    out = torch.full((3, 8 * D + 8), 7.0, device="cuda")
    y = out[:, :8 * D].unflatten(1, (8, D))
    ws = torch.full((_lib.load().qd_paged_attn_decode_workspace_bytes(3, 8),), 255, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = R.paged_attn_decode(q, k, v, table, n, scale=0.25, y=y, workspace=ws, stream=stream)
    stream.synchronize()
    want, tol = plain_attention(torch, q, k, v, table, n, [1] * 3, 0, 0, 0.25, "f32", "f16")
    close(torch, got, want, tol)
    assert got.data_ptr() == out.data_ptr() and bool((out[:, 8 * D:] == 7).all())
    flat = R.paged_attn_decode(q.reshape(3, -1), k, v, table[:, :12], n, scale=0.25)   # rows of a wider table
    assert torch.equal(flat.view(3, 8, D), got)
    with pytest.raises(ValueError):
        R.paged_attn_decode(q, k, v, table, n, workspace=ws[:16])


@pytest.mark.gpu
def test_decode_is_the_same_every_time_and_replays_with_new_lengths():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [900, 33, 2500, 1]
    k, v, table, n = make_cache(torch, lens, 16, 2, "f16")
    q = torch.randn(4, 16, D, device="cuda")
    first = R.paged_attn_decode(q, k, v, table, n).clone()
    for _ in range(3):
        assert torch.equal(R.paged_attn_decode(q, k, v, table, n), first)
    # two graphs of the same tensors with workspaces of their own
    ws = [torch.empty(_lib.load().qd_paged_attn_decode_workspace_bytes(4, 16), dtype=torch.uint8, device="cuda")
          for _ in range(2)]
    y = [torch.zeros_like(q) for _ in range(2)]
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            R.paged_attn_decode(q, k, v, table, n, y=y[i], workspace=ws[i], window=1000 * i)
        graphs.append(graph)
    for shorter in ([900, 33, 2500, 1], [1, 32, 1200, 0]):
        n.copy_(torch.tensor(shorter, dtype=torch.int32))
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want, tol = plain_attention(torch, q, k, v, table, n, [1] * 4, 1000 * i, 0, D ** -0.5, "f32", "f16")
            close(torch, y[i], want, tol)


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_left_out_and_flagged():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [100, 40], 16, 2, "f16")
    q = torch.randn(2, 4, D, device="cuda")
    table[0, 2] = k.shape[0]       # one past the pool: positions 32..47 of sequence 0 are left out
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode(q, k, v, table, n, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_PAGE
    keep = torch.cat([torch.arange(32), torch.arange(48, 100)]).cuda()
    pg = table[0].long()[keep // 16]
    kk, vv = (x[pg, :, keep % 16].double().repeat_interleave(2, 1) for x in (k, v))
    w = torch.softmax(torch.einsum("hd,jhd->hj", q[0].double(), kk) / math.sqrt(D), -1)
    assert float((y[0].double() - torch.einsum("hj,jhd->hd", w, vv)).abs().max()) < 1e-4
    status.zero_()
    y = R.paged_attn_prompt(q, k, v, table, n, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), status=status)
    assert int(status) == _lib.QD_PAGED_BAD_PAGE
    assert float((y[0].double() - torch.einsum("hj,jhd->hd", w, vv)).abs().max()) < 1e-4
    # a length beyond the table is cut to the table
    status.zero_()
    table[0, 2] = table[0, 1]
    n[0] = 10 ** 9
    y = R.paged_attn_decode(q, k, v, table, n, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_LENGTH and bool(torch.isfinite(y).all())
    # a negative length holds nothing
    status.zero_()
    n[0] = -3
    y = R.paged_attn_decode(q, k, v, table, n, status=status)
    assert bool((y[0] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("pages", [0, 4])
def test_sequences_without_a_single_usable_page(io, cache, pages):
    """No pool, or entries that name no page of it: zeros, flagged, and nothing is written."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    T = _types(torch)
    k, v = (torch.full((pages, 2, 64, D), math.nan, dtype=T[cache], device="cuda") for _ in "kv")
    table = torch.full((2, 3), pages, dtype=torch.int32, device="cuda")
    n = torch.tensor([150, 2], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 140, 142], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.randn(142, 4, D, device="cuda").to(T[io])
    for call in (lambda: R.paged_attn_prompt(q, k, v, table, n, starts, status=status),
                 lambda: R.paged_attn_decode(q[:2], k, v, table, n, status=status)):
        assert bool((call() == 0).all()) and int(status) == _lib.QD_PAGED_BAD_PAGE
        status.zero_()
    R.paged_append(torch.randn(142, 8 * D, device="cuda"), k, v, table, n, None, None, 4, q_starts=starts, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_PAGE and bool(torch.isnan(k).all()) and bool(torch.isnan(v).all())


@pytest.mark.gpu
@pytest.mark.parametrize("length,bits", [(0, 0), (-1, _lib.QD_PAGED_BAD_LENGTH), (-2 ** 31, _lib.QD_PAGED_BAD_LENGTH),
                                         (2, _lib.QD_PAGED_BAD_LENGTH), (3, 0), (40, 0), (48, 0),
                                         (49, _lib.QD_PAGED_BAD_LENGTH), (2 ** 31 - 1, _lib.QD_PAGED_BAD_LENGTH)])
def test_lengths_that_have_no_place_are_flagged(length, bits):
    """Three new tokens of a sequence in a table of 48 positions: the rows at positions below 0 give zeros."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [48, 48], 16, 2, "f16")
    q = torch.randn(5, 4, D, device="cuda")
    starts = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    n.copy_(torch.tensor([length, 48], dtype=torch.int32))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_prompt(q, k, v, table, n, starts, status=status)
    assert int(status) == bits
    before = min(3, max(0, 3 - length))
    assert bool((y[:before] == 0).all()) and bool((y[before:3] != 0).any(-1).all())
    other = R.paged_attn_prompt(q[3:], k, v, table[1:], n[1:], torch.tensor([0, 2], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[3:], other)
    status.zero_()
    y = R.paged_attn_decode(q[:2], k, v, table, n, status=status)
    assert int(status) == (bits if length != 2 else 0)
    assert bool((y[0] == 0).all()) == (length <= 0)


# ---- attention of prompt chunks ------------------------------------------------------------

CHUNKS = [([8], [8]), ([1], [1]), ([130], [130]), ([1, 0, 70, 5], [900, 40, 70, 6]), ([300, 17], [513, 1100]),
          ([33] * 9, [33 + 40 * i for i in range(9)]), ([700], [1000]), ([0, 3, 0], [0, 3, 9])]


def run_prompt(torch, new, totals, heads, page, io, cache, window, sinks, pad=3, fill=math.nan):
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, totals, page, heads[1], cache, seed=sum(new), fill=fill)
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    rows = sum(new) + pad
    q = (torch.randn(rows, heads[0], D, device="cuda") * 1.5).to(_types(torch)[io])
    q[sum(new):] = math.nan
    y = torch.full_like(q, 5.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = R.paged_attn_prompt(q, k, v, table, n, starts, window=window, sinks=sinks, y=y, status=status)
    assert bool((got[sum(new):] == 5.0).all()), "padding rows were written"
    assert int(status) == 0
    want, tol = plain_attention(torch, q, k, v, table, n, new, window, sinks, D ** -0.5, io, cache)
    close(torch, got[:sum(new)], want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", CHUNKS, ids=lambda c: f"{len(c[0])}x{max(c[0])}of{max(c[1])}")
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
def test_prompt_attention(chunk, heads, io, cache):
    torch = _cuda()
    run_prompt(torch, *chunk, heads, [16, 64, 128, 256][(len(chunk[0]) + heads[0]) % 4], io, cache, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (128, 4), (129, 130), (300, 1), (64, 700), (5000, 4)])
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_prompt_window_and_sinks(window, sinks, io, cache):
    torch = _cuda()
    run_prompt(torch, [400, 1, 70], [900, 300, 70], (8, 2), 16, io, cache, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16")])
def test_long_prompt_over_many_key_tiles(io, cache):
    """Enough rows that the keys are not split over CTAs, and up to 15 tiles of them in one row's sums."""
    torch = _cuda()
    run_prompt(torch, [1500, 90], [1900, 1800], (16, 8), 32, io, cache, 0, 0)


def many_chunks():
    rng = random.Random(11)
    new = [rng.choice([0, 1, 2, 33, 64, 127, 128, 129, 200]) for _ in range(60)]
    return new, [n + rng.choice([0, 0, 5, 100, 700]) for n in new]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
@pytest.mark.parametrize("heads", [(4, 4), (8, 4), (28, 4)], ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
def test_prompt_of_more_blocks_than_run_at_once(io, cache, heads, window, sinks):
    torch = _cuda()
    run_prompt(torch, *many_chunks(), heads, 16, io, cache, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_prompt_of_many_blocks_some_with_nothing_to_see(io):
    """Sequences whose length says that nothing was appended give zeros; the others' rows stay as they are,
    to the bit, and in every one of several runs."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    new, totals = many_chunks()
    k, v, table, n = make_cache(torch, totals, 32, 4, "f16")
    starts = torch.tensor([sum(new[:b]) for b in range(61)], dtype=torch.int32, device="cuda")
    q = torch.randn(sum(new), 8, D, device="cuda").to(_types(torch)[io])
    want = R.paged_attn_prompt(q, k, v, table, n, starts)
    none = n.clone()
    none[::3] = 0
    hit = torch.zeros(sum(new), dtype=torch.bool, device="cuda")
    for b in range(0, 60, 3):
        hit[sum(new[:b]):sum(new[:b + 1])] = True
    for _ in range(5):
        got = R.paged_attn_prompt(q, k, v, table, none, starts)
        assert bool((got[hit] == 0).all()) and torch.equal(got[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_captured_prompts_follow_their_lengths_on_two_streams(io):
    """A captured call over padded rows, replayed with other chunks, beside a second one on its own stream."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    rows, graphs = 6000, []
    for seed in (0, 1):
        new, totals = many_chunks()
        k, v, table, n = make_cache(torch, totals, 16, 4, "f16", seed=seed)
        starts = torch.tensor([sum(new[:b]) for b in range(61)], dtype=torch.int32, device="cuda")
        q = torch.randn(rows, 8, D, device="cuda").to(_types(torch)[io])
        y = torch.zeros_like(q)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        R.paged_attn_prompt(q, k, v, table, n, starts, y=y)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            R.paged_attn_prompt(q, k, v, table, n, starts, y=y)
        graphs.append((stream, graph, q, k, v, table, n, starts, y, new, totals))
    for turn in range(4):
        for stream, graph, q, k, v, table, n, starts, y, new, totals in graphs:
            some = [c if (b + turn) % 4 else 0 for b, c in enumerate(new)]
            starts.copy_(torch.tensor([sum(some[:b]) for b in range(61)], dtype=torch.int32))
            n.copy_(torch.tensor([t - c + s for t, c, s in zip(totals, new, some)], dtype=torch.int32))
            y.fill_(7.0)
        torch.cuda.synchronize()
        for stream, graph, *_ in graphs:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for stream, graph, q, k, v, table, n, starts, y, new, totals in graphs:
            want = R.paged_attn_prompt(q, k, v, table, n, starts, y=torch.full_like(y, 7.0))
            used = int(starts[-1])
            assert torch.equal(y, want) and bool((y[used:] == 7.0).all()) and not bool((y[:used] == 7.0).any())


@pytest.mark.gpu
def test_prompt_equals_decode_for_single_tokens():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [70, 1, 515, 128]
    k, v, table, n = make_cache(torch, lens, 32, 8, "f16")
    q = torch.randn(4, 16, D, device="cuda")
    starts = torch.arange(5, dtype=torch.int32, device="cuda")
    a, b = R.paged_attn_prompt(q, k, v, table, n, starts), R.paged_attn_decode(q, k, v, table, n)
    _, tol = plain_attention(torch, q, k, v, table, n, [1] * 4, 0, 0, D ** -0.5, "f32", "f16")
    close(torch, a, b.double(), 2 * tol)


@pytest.mark.gpu
def test_a_causal_future_of_large_values_does_not_reach_the_past():
    """Rows before a token see nothing of its K and V, however large these are."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    new = [150]
    k, v, table, n = make_cache(torch, new, 16, 1, "f16")
    starts = torch.tensor([0, 150], dtype=torch.int32, device="cuda")
    q = torch.randn(150, 2, D, device="cuda").half()
    before = R.paged_attn_prompt(q, k, v, table, n, starts).clone()
    pg = table[0].long()
    for p in range(140, 150):
        k[pg[p // 16], :, p % 16] = 60000.0
        v[pg[p // 16], :, p % 16] = -60000.0
    after = R.paged_attn_prompt(q, k, v, table, n, starts)
    assert torch.equal(before[:140], after[:140]) and bool(torch.isfinite(after).all())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-20, 1e-4, 1.0, 1e5, 1e20])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_f32_queries_of_any_size(size, sign, cache):
    """The scores are ordinary, whatever share of them q and the scale hold: f32 queries keep their accuracy far
    outside f16's range, rows of every size in one call, a few large elements in a row among them."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    new, totals = [300, 3], [330, 200]
    k, v, table, n = make_cache(torch, totals, 32, 2, cache)
    q = torch.randn(303, 8, D, device="cuda") * 1.5
    q[::3] *= 0.01
    q[1::5, :, 7] *= 300.0
    q *= size
    scale = sign * D ** -0.5 / size
    y = R.paged_attn_prompt(q, k, v, table, n, torch.tensor([0, 300, 303], dtype=torch.int32, device="cuda"), scale=scale)
    want, tol = plain_attention(torch, q, k, v, table, n, new, 0, 0, scale, "f32", cache)
    close(torch, y, want, tol)
    y = R.paged_attn_decode(q[:2], k, v, table, n, scale=scale)
    want, tol = plain_attention(torch, q[:2], k, v, table, n, [1, 1], 0, 0, scale, "f32", cache)
    close(torch, y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_zero_and_large_queries_and_large_scales(io):
    """Zeros weigh all keys alike; f16 queries times a large scale leave f16's range, not f32's."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [90, 70], 16, 2, "f16")
    q = (torch.randn(2, 4, D, device="cuda") * 1.5e4).clamp(-6e4, 6e4).to(_types(torch)[io])
    q[0] = 0.0
    starts = torch.arange(3, dtype=torch.int32, device="cuda")
    for y in (R.paged_attn_decode(q, k, v, table, n, scale=20.0), R.paged_attn_prompt(q, k, v, table, n, starts, scale=20.0)):
        want, tol = plain_attention(torch, q[:1], k, v, table[:1], n[:1], [1], 0, 0, 20.0, io, "f16")
        close(torch, y[:1], want, tol)
        # scores of 1e7 and more, thousands apart: one key has all the weight
        j = torch.arange(70, device="cuda")
        kk, vv = (x[table[1].long()[j // 16], :, j % 16].double().repeat_interleave(2, 1) for x in (k, v))
        best = torch.einsum("hd,jhd->hj", q[1].double(), kk).argmax(-1)
        want = vv[best, torch.arange(4, device="cuda")]
        # The scores, in units of 1e7 log2 e, leave the maximum's f32 rounding (half of 2) in the exponent, so the one
        # weight is no power of two: with 16-bit queries it is rounded to f16 once (half a step, 2^-11) where
        # its sum is not; then the sum, a division and y's own rounding.
        weight = 2.0 ** -11 if io == "f16" else 2.0 ** -21
        close(torch, y[1], want, (weight + HALF_STEP[io] + 2.0 ** -22) * want.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(2, 2), (3, 1), (16, 2)], ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("io,cache", [("f16", "f16"), ("f32", "f16"), ("f32", "bf16")])
def test_how_far_a_v_row_that_is_not_finite_reaches(heads, io, cache):
    """A NaN or an infinity in one visible V row: rows that see it, and no row 256 tokens * heads from those."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    new, at, window = 1400, 700, 40
    k, v, table, n = make_cache(torch, [new], 16, heads[1], cache)
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    q = torch.randn(new, heads[0], D, device="cuda").to(_types(torch)[io])
    want = R.paged_attn_prompt(q, k, v, table, n, starts, window=window)
    reach = -(-256 // (heads[0] // heads[1]))
    p = torch.arange(new, device="cuda")
    sees = (p >= at) & (p < at + window)
    near = (p > at - reach) & (p < at + window + reach)
    for bad in (math.nan, math.inf):
        v2 = v.clone()
        v2[table[0, at // 16].long(), 0, at % 16, 5] = bad
        y = R.paged_attn_prompt(q, k, v2, table, n, starts, window=window)
        gone = ~torch.isfinite(y)
        assert bool(gone[sees, :heads[0] // heads[1], 5].all())
        assert torch.equal(y[~near], want[~near]) and not bool(gone[:, heads[0] // heads[1]:].any())
        gone[..., 5] = False
        assert not bool(gone.any())


# ---- the accuracy of f32 queries ---------------------------------------------------------------

def two_keys(torch, n, cache):
    """n pairs of keys, seen by one query each, whose scores are two elements of q: (q, keys, values, y in 64 bits). With
    the scale ln 2 the factor of the scores is 1 in f32, so a kernel that keeps all of q has their exact difference."""
    T = _types(torch)[cache]
    g = torch.Generator().manual_seed(n)
    a = 24 + 8 * torch.rand(n, 2, generator=g)
    b = a + 0.7 * torch.randn(n, 2, generator=g)
    q = torch.zeros(n, 2, D)
    q[..., 0], q[..., 1] = a, b
    k = torch.zeros(2, D)
    k[0, 0] = k[1, 1] = 1.0
    v = torch.ones(2, D)
    v[1] = -1.0
    return q, k.to(T), v.to(T), torch.tanh((a.double() - b.double()) * math.log(2) / 2)


def f32_tolerance(cache):
    """Of |w0 - w1| / (w0 + w1): the exponential (2^-22), at most 6 truncated additions of products (2^-23 each), as
    many roundings in f32 of sums, joins and the division (2^-24). Two f16 hold 22 bits: half a step of 2^-22 of scores
    up to 34 (in units of log2) and of the weights. Three bf16 hold all 24."""
    return 2.0 ** -22 + 6 * 2.0 ** -23 + 6 * 2.0 ** -24 + (math.log(2) * 34 * 2.0 ** -23 + 2.0 ** -22 if cache == "f16" else 0)


def parts(torch, x, n, T):
    """x as a sum of n rounded parts."""
    out = torch.zeros_like(x)
    for _ in range(n):
        out = out + (x - out).to(T).double()
    return out


def test_the_tolerance_of_f32_queries_tells_two_bf16_from_three():
    torch = pytest.importorskip("torch")
    q, _, _, want = two_keys(torch, 600, "bf16")
    a, b = q[..., 0].double(), q[..., 1].double()
    for q_parts, w_parts, passes in ((3, 3, True), (2, 3, False), (3, 2, False)):
        x, y = parts(torch, a, q_parts, torch.bfloat16), parts(torch, b, q_parts, torch.bfloat16)
        m = torch.maximum(x, y)
        w0, w1 = torch.exp2(x - m + 7), torch.exp2(y - m + 7)
        got = (parts(torch, w0, w_parts, torch.bfloat16) - parts(torch, w1, w_parts, torch.bfloat16)) / (w0 + w1)
        assert (float((got - want).abs().max()) <= f32_tolerance("bf16")) == passes


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_f32_queries_keep_their_bits(cache):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    n = 600
    q, keys, values, want = (x.cuda() for x in two_keys(torch, n, cache))
    # decode: n sequences of two positions
    k, v, table, lens = make_cache(torch, [2] * n, 16, 1, cache)
    pg = table[:, 0].long()
    k[pg, 0, :2], v[pg, 0, :2] = keys, values
    y = R.paged_attn_decode(q, k, v, table, lens, scale=math.log(2))
    close(torch, y, want[..., None].expand(n, 2, D), torch.full((1,), f32_tolerance(cache), device="cuda"))
    # prompt: every row sees the sink and itself
    k, v, table, lens = make_cache(torch, [n + 1], 16, 1, cache)
    pg = table[0].long()
    k[pg, 0], v[pg, 0] = keys[1], values[1]
    k[pg[0], 0, 0], v[pg[0], 0, 0] = keys[0], values[0]
    y = R.paged_attn_prompt(q, k, v, table, lens, torch.tensor([0, n], dtype=torch.int32, device="cuda"), window=1,
                            sinks=1, scale=math.log(2))
    close(torch, y, want[..., None].expand(n, 2, D), torch.full((1,), f32_tolerance(cache), device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_long_rows_of_f32_queries_do_not_drift(cache):
    """Rows over 4000 keys with positive values, where every truncated addition of the tensor cores drifts the same
    way. Scores of one product: off by its roundings, 3 * 2^-23 of scores up to 4, and (f16) half a step of 22 bits of
    q. Weights: the exponential of arguments up to 16 (2^-21, 2^-22), their parts (2^-22). Sums: between two moves out
    of TMEM at most 4 tiles * 8 steps * 3 parts, each of which drops up to 2^-23 of a sum that is half grown on the
    average; then 8 moves, the sum of weights (32 chains of additions a tile) and the division, 2^-24 each."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    new, total = 600, 4000      # 80 row tiles or more: their keys are not split over CTAs
    k, v, table, lens = make_cache(torch, [total], 32, 16, cache)
    g = torch.Generator(device="cuda").manual_seed(1)
    k[..., 1:] = 0
    k[..., 0] = torch.rand(k.shape[:3], generator=g, device="cuda").to(k.dtype) * 2 - 1
    v.copy_((1 + torch.rand(v.shape, generator=g, device="cuda")).to(v.dtype))
    q = torch.zeros(new, 32, D, device="cuda")
    q[..., 0] = 4 * torch.rand(new, 32, generator=g, device="cuda")
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    y = R.paged_attn_prompt(q, k, v, table, lens, starts, scale=1.0)
    want, _ = plain_attention(torch, q, k, v, table, lens, [new], 0, 0, 1.0, "f32", cache)
    weights = 2 * (4 * 3 * 2.0 ** -23 + 4 * (2.0 ** -23 if cache == "f16" else 0) + 2.0 ** -21 + 2.0 ** -22 + 2.0 ** -22)
    sums = 4 * 8 * (3 if cache == "bf16" else 2) / 2 * 2.0 ** -23 + (8 + 32 + 2) * 2.0 ** -24
    close(torch, y, want, (weights + sums) * want)


# ---- norm + rotation + append ----------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("io,cache,out", [("f32", "f16", "f32"), ("bf16", "bf16", "bf16"), ("f16", "f16", "f16"),
                                          ("f32", "bf16", "bf16"), ("f32", "f16", "f16")])
@pytest.mark.parametrize("new,totals", [([1], [9]), ([1, 1, 1], [5, 1, 700]), ([40, 0, 3, 129], [40, 7, 300, 129]),
                                        ([1] * 200, list(range(1, 201)))], ids=["one", "three", "ragged", "many"])
@pytest.mark.parametrize("heads", [(16, 8), (5, 1), (0, 2)], ids=lambda h: f"{h[0]}q{h[1]}kv")
def test_append(io, cache, out, new, totals, heads):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    T = _types(torch)
    H, kvh = heads
    k, v, table, n = make_cache(torch, totals, 16, kvh, cache)
    rows, pad = sum(new), 2
    qkv = torch.randn(rows + pad, (H + 2 * kvh) * D + 24, device="cuda").to(T[io])[:, :(H + 2 * kvh) * D]
    qn, kn = torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda") + 0.5
    angle = torch.rand(max(totals), 64, device="cuda") * 6.28
    cos, sin = angle.cos(), angle.sin()
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    q_out = torch.full((rows + pad, H * D), 3.0, device="cuda").to(T[out])
    k0, v0 = k.clone(), v.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    R.paged_append(qkv, k, v, table, n, cos, sin, H, q_norm=qn, k_norm=kn, q_starts=starts, q_out=q_out, status=status)
    assert int(status) == 0 and bool((q_out[rows:] == 3).all())
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(t - m, t) for m, t in zip(new, totals)]).cuda()
    x = qkv[:rows].double().unflatten(1, (-1, D))

    def turned(h, w):
        h = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        a, b = h[..., :64], h[..., 64:]
        # 128 squares (at most 9 roundings, halved by the root), the root (2 steps), two
        # products with the weight and two with the rotation: under 16 half steps of f32
        tol = 16 * 2.0 ** -24 * torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1), tol

    want, tol = turned(x[:, :H], qn)
    close(torch, q_out[:rows].unflatten(1, (-1, D)) if H else q_out[:rows].view(rows, 0, D), want,
          tol + HALF_STEP[out] * want.abs() + 2.0 ** -25)
    pg = table[seq].long().gather(1, (pos // 16)[:, None])[:, 0]
    want, tol = turned(x[:, H:H + kvh], kn)
    close(torch, k[pg, :, pos % 16], want, tol + HALF_STEP[cache] * want.abs() + 2.0 ** -25)
    assert torch.equal(v[pg, :, pos % 16], qkv[:rows].float().unflatten(1, (-1, D))[:, H + kvh:].to(T[cache]))
    untouched = torch.ones(k.shape[0], k.shape[2], dtype=torch.bool, device="cuda")
    untouched[pg, pos % 16] = False
    assert torch.equal(k.transpose(1, 2)[untouched], k0.transpose(1, 2)[untouched])
    assert torch.equal(v.transpose(1, 2)[untouched], v0.transpose(1, 2)[untouched])


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 2, 31, 32, 33, 64, 65, 1023, 1024, 1025, 4096])
def test_append_finds_the_rows_of_any_number_of_sequences(batch):
    """Ragged chunks, empty ones among them, behind which the buffer ends: padding rows are not read."""
    torch = _cuda()
    rng = random.Random(batch)
    new = [rng.choice([0, 0, 1, 2, 3]) for _ in range(batch)]
    new[batch // 2] = 2
    rows, pad = sum(new), 37
    k, v, table, n = make_cache(torch, [m + rng.randrange(9) for m in new], 16, 1, "f16")
    starts = torch.tensor([sum(new[:b]) for b in range(batch + 1)], dtype=torch.int32, device="cuda")
    qkv = torch.randn(rows, 4 * D, device="cuda")              # the last rows + pad .. rows of it do not exist
    out = torch.full((rows + pad, 2 * D), 9.0, device="cuda")
    kv = _kv(k=k.data_ptr(), v=v.data_ptr(), num_pages=k.shape[0], kv_heads=1, batch=batch,
             block_table=table.data_ptr(), table_width=table.shape[1], table_stride=table.shape[1],
             seq_lens=n.data_ptr())
    rc = _lib.load().qd_paged_append(kv, qkv.data_ptr(), _lib.QD_KV_F32, 4 * D, rows + pad, starts.data_ptr(), 2, None,
                                     None, 1e-6, None, None, 0, 0, out.data_ptr(), _lib.QD_KV_F32, 2 * D,
                                     torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.QD_OK
    assert torch.equal(out[:rows], qkv[:, :2 * D]) and bool((out[rows:] == 9.0).all())
    seq = torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(int(t) - m, int(t)) for m, t in zip(new, n.tolist())]).cuda()
    pg = table[seq].long().gather(1, (pos // 16)[:, None])[:, 0]
    assert torch.equal(k[pg, 0, pos % 16], qkv[:, 2 * D:3 * D].half())
    assert torch.equal(v[pg, 0, pos % 16], qkv[:, 3 * D:].half())


@pytest.mark.gpu
def test_append_in_place_without_norm_or_rotation_and_wider_table_rows():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [3, 20], 16, 2, "f16")
    qkv = torch.randn(2, 8 * D, device="cuda")
    x = qkv.clone()
    q = R.paged_append(qkv, k, v, table, n, None, None, 4, q_out=qkv[:, :4 * D])      # plain append, in place
    assert torch.equal(q, x[:, :4 * D])
    assert torch.equal(k[table[1, 1].long(), :, 3], x[1, 4 * D:6 * D].view(2, D).half())
    # rows of the table 128 apart, as the reference reads it (position p at row 2p)
    cos, sin = torch.rand(40, 64, device="cuda"), torch.rand(40, 64, device="cuda")
    a = R.paged_append(x, k, v, table, n, cos, sin, 4, rope_stride=128)
    b = R.paged_append(x, k, v, table, n, cos[::2].contiguous(), sin[::2].contiguous(), 4)
    assert torch.equal(a, b)
    q2 = R.paged_append(x, k, v, table, n, cos, sin, 4, rope_stride=128, q_out=x[:, :4 * D])
    assert torch.equal(q2, a)


@pytest.mark.gpu
def test_append_flags_what_has_no_place():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [16, 16, 16, 16], 16, 1, "f16")
    n.copy_(torch.tensor([17, 0, 5, 9]))       # beyond the table; a new token at position -1; fine; bad page below
    table[3, 0] = -1
    k0 = k.clone()
    cos = torch.rand(4, 64, device="cuda")       # tables end before position 4
    x = torch.randn(4, 4 * D, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    R.paged_append(x, k, v, table, n, cos, cos, 2, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_LENGTH and torch.equal(k, k0)
    status.zero_()
    R.paged_append(x[3:], k, v, table[3:], n[3:], None, None, 2, status=status)
    assert int(status) == _lib.QD_PAGED_BAD_PAGE and torch.equal(k, k0)


@pytest.mark.gpu
def test_rotation_tables_that_are_not_rows_by_position_are_refused():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [5, 9], 16, 1, "f16")
    x = torch.randn(2, 4 * D, device="cuda")
    rows = torch.rand(20, 64, device="cuda")
    wide = torch.cat([rows, rows], 1).contiguous()
    want = R.paged_append(x, k, v, table, n, rows, rows, 2)
    for cos, sin in ((wide, wide), (rows.reshape(-1), rows.reshape(-1)), (rows[:, None], rows[:, None])):
        assert torch.equal(R.paged_append(x, k, v, table, n, cos, sin, 2), want)
    one = torch.as_strided(wide, (1, 64), (128, 1))       # one row: its stride says nothing
    got = R.paged_append(x[:1], k, v, table[:1], torch.ones_like(n[:1]), one, one, 2)
    assert torch.equal(got, R.paged_append(x[:1], k, v, table[:1], torch.ones_like(n[:1]), rows, rows, 2))
    half = rows[:, :32].contiguous()
    for cos, sin in ((wide, rows), (rows, wide), (half, half), (rows[None], rows[None]), (rows, rows[:10])):
        with pytest.raises(ValueError, match="positions"):
            R.paged_append(x, k, v, table, n, cos, sin, 2)
    assert torch.equal(R.paged_append(x, k, v, table, n, rows, rows[:10], 2, rope_stride=64), want)


@pytest.mark.gpu
def test_a_scale_below_float32_is_not_the_default():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [5, 9], 16, 1, "f16")
    q = torch.randn(2, 2, D, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for call in (lambda s: R.paged_attn_decode(q, k, v, table, n, scale=s),
                 lambda s: R.paged_attn_prompt(q, k, v, table, n, starts, scale=s)):
        with pytest.raises(ValueError, match="scale"):
            call(1e-60)
        mean = v[table[0, 0].long(), 0, :5].double().mean(0)      # every key alike
        close(torch, call(1e-40)[0], mean.expand(2, D), 2.0 ** -20 * v[table[0, 0].long(), 0, :5].double().abs().mean(0))


# ---- the step as it is used -------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("cache,window", [("f16", 0), ("bf16", 24)])
def test_prompt_then_decoding_steps_over_one_cache(cache, window):
    """Three sequences: their prompts in two ragged chunks, then single tokens, then a draw:
    the attention outputs equal those of a 64-bit evaluation over the rows that the appends
    left in the cache, and the tokens are the definition's."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    torch.manual_seed(5)
    H, kvh, page, sinks = 8, 2, 16, 4
    T = _types(torch)[cache]
    k, v = (torch.full((40, kvh, page, D), math.nan, device="cuda", dtype=T) for _ in "kv")
    table = torch.randperm(40, device="cuda")[:36].to(torch.int32).view(3, 12)
    a = torch.outer(torch.arange(192, device="cuda").double(), 1e6 ** (-torch.arange(64, device="cuda").double() / 64))
    cos, sin = a.cos().float(), a.sin().float()
    qn, kn = torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda") + 0.5
    held = torch.zeros(3, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    head = torch.randn(H * D, 997, device="cuda") * 0.05
    for new in ([70, 3, 33], [41, 1, 0], [1, 1, 1], [1, 1, 1]):
        held += torch.tensor(new, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32, device="cuda")
        qkv = torch.randn(sum(new), (H + 2 * kvh) * D, device="cuda")
        q = R.paged_append(qkv, k, v, table, held, cos, sin, H, q_norm=qn, k_norm=kn, q_starts=starts, status=status)
        q = q.view(-1, H, D)
        if max(new) > 1:
            y = R.paged_attn_prompt(q, k, v, table, held, starts, window=window, sinks=sinks, status=status)
        else:
            y = R.paged_attn_decode(q, k, v, table, held, window=window, sinks=sinks, status=status)
        want, tol = plain_attention(torch, q, k, v, table, held, new, window, sinks, D ** -0.5, "f32", cache)
        close(torch, y, want, tol)
    logits = y.reshape(3, -1) @ head
    ids, logp = R.sample_rows(logits, torch.tensor([0.1, 0.5, 0.9], device="cuda"),
                              temperature=torch.tensor([0.0, 1.0, 0.7], device="cuda"),
                              top_k=torch.tensor([0, 1, 50], dtype=torch.int32, device="cuda"))
    assert ids[:2].tolist() == logits[:2].argmax(-1).tolist()
    w = torch.softmax(logits[2].double().topk(50).values / 0.7, 0)
    rank = int((w.cumsum(0) <= 0.9).sum())
    assert int(ids[2]) == int(logits[2].topk(50).indices[rank]) and abs(float(logp[2]) - math.log(float(w[rank]))) < 1e-5
    assert int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_offsets_beyond_32_bits(io):
    """Pools of 5.2 GB whose used pages lie at both ends, and rows 4.4 GB apart."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    pages, kvh, page, H = 40000, 8, 64, 16
    T = _types(torch)[io]
    k, v = (torch.empty(pages, kvh, page, D, dtype=torch.float16, device="cuda") for _ in "kv")
    small_k, small_v, small, n = make_cache(torch, [300, 131], page, kvh, "f16")
    used = torch.unique(small[small >= 0]).long()
    far = torch.where(used % 2 == 0, pages - 1 - used, used)
    k[far], v[far] = small_k[used], small_v[used]
    table = small.clone()
    for a, b in zip(used.tolist(), far.tolist()):
        table[small == a] = b
    wide = (2 ** 32 + 2 ** 28) // T.itemsize          # elements between two rows
    store = torch.empty(wide + 64 * D, dtype=T, device="cuda")
    qkv = store.as_strided((2, (H + 2 * kvh) * D), (wide, 1))
    qkv.copy_(torch.randn(2, (H + 2 * kvh) * D, device="cuda"))
    near = qkv.clone()
    want = R.paged_append(near, small_k, small_v, small, n, None, None, H)
    got = R.paged_append(qkv, k, v, table, n, None, None, H, q_out=qkv[:, :H * D])
    assert torch.equal(got, want) and torch.equal(k[far], small_k[used]) and torch.equal(v[far], small_v[used])
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    y = store.as_strided((2, H, D), (wide, D, 1), (H + 2 * kvh) * D)
    big = R.paged_attn_decode(got.unflatten(1, (H, D)), k, v, table, n, y=y)
    assert torch.equal(big, R.paged_attn_decode(want.unflatten(1, (H, D)), small_k, small_v, small, n))
    big = R.paged_attn_prompt(got.unflatten(1, (H, D)), k, v, table, n, starts, y=y)
    assert torch.equal(big, R.paged_attn_prompt(want.unflatten(1, (H, D)), small_k, small_v, small, n, starts))
    u = torch.rand(2, device="cuda")
    ids, logp = R.sample_rows(qkv, u)
    want_ids, want_logp = R.sample_rows(qkv.clone(), u)
    assert torch.equal(ids, want_ids) and torch.equal(logp, want_logp)


@pytest.mark.gpu
def test_a_thread_without_a_cuda_call_before_it():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [40, 7], 16, 2, "f16")
    q = torch.randn(2, 4, D, device="cuda")
    starts = torch.arange(3, dtype=torch.int32, device="cuda")
    u = torch.rand(2, device="cuda")
    calls = [lambda: R.paged_attn_prompt(q, k, v, table, n, starts), lambda: R.paged_attn_decode(q, k, v, table, n),
             lambda: R.paged_append(q.view(1, 8 * D), k, v, table[:1], n[:1], None, None, 4),
             lambda: R.sample_rows(q.view(2, -1), u)[0]]
    for call in calls:
        want, got = call(), []
        thread = threading.Thread(target=lambda: got.append(call()))
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want)


@pytest.mark.gpu
def test_calls_from_many_threads_at_once():
    """Eight threads with streams, outputs and workspaces of their own, every entry among them; the C ABI, under
    which Python's threads do run together, in a process that has made no call before."""
    _cuda()
    code = textwrap.dedent("""
        import threading, torch
        from kernel_optimization_webgpu_b200 import _lib, runtime as R
        L = _lib.load()
        torch.manual_seed(0)
        lens = [700, 33, 64, 129]
        per = -(-max(lens) // 32)
        k, v = (torch.randn(4 * per, 2, 32, 128, device="cuda").half() for _ in "kv")
        table = torch.randperm(4 * per, device="cuda").to(torch.int32).view(4, per)
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        kv = _lib.QdPagedKv(k.data_ptr(), v.data_ptr(), 0, 4 * per, 32, 2, 128, 4, table.data_ptr(), per, per, n.data_ptr(), None)
        starts = torch.tensor([0, 300, 310, 311, 400], dtype=torch.int32, device="cuda")
        q = torch.randn(400, 8, 128, device="cuda")
        logits, u = torch.randn(4, 5000, device="cuda"), torch.rand(4, device="cuda")
        outs, codes, gate = [], [], threading.Barrier(8)
        for i in range(8):
            outs.append([torch.zeros(400, 8, 128, device="cuda"), torch.zeros(4, 8, 128, device="cuda"),
                         torch.zeros(4, dtype=torch.int32, device="cuda"), torch.cuda.Stream(),
                         torch.empty(L.qd_paged_attn_prompt_workspace_bytes(4, 400, 8, 2, 1), dtype=torch.uint8, device="cuda"),
                         torch.empty(L.qd_paged_attn_decode_workspace_bytes(4, 8), dtype=torch.uint8, device="cuda")])
        torch.cuda.synchronize()
        def work(i):
            yp, yd, ids, stream, wp, wd = outs[i]
            s = stream.cuda_stream
            gate.wait()
            for _ in range(20):
                codes.append(L.qd_paged_attn_prompt(kv, q.data_ptr(), 1, 1024, 400, starts.data_ptr(), 8, 0, 0, 0.0,
                                                    yp.data_ptr(), 1024, wp.data_ptr(), s))
                codes.append(L.qd_paged_attn_decode(kv, q.data_ptr(), 1, 1024, 8, 0, 0, 0.0, yd.data_ptr(), 1024,
                                                    wd.data_ptr(), s))
                codes.append(L.qd_sample_rows(logits.data_ptr(), 1, 4, 5000, 5000, None, None, None, None, u.data_ptr(),
                                              ids.data_ptr(), None, s))
        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        for t in threads: t.start()
        for t in threads: t.join()
        torch.cuda.synchronize()
        want = (R.paged_attn_prompt(q, k, v, table, n, starts), R.paged_attn_decode(q[:4], k, v, table, n),
                R.sample_rows(logits, u)[0])
        assert codes == [0] * 480, codes
        print(all(torch.equal(a, b) for o in outs for a, b in zip(o, want)))
    """)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=_lib._build.ROOT)
    assert res.returncode == 0 and res.stdout.split() == ["True"], res.stderr
