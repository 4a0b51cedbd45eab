"""Local attention and its position bias on the GPU against the float64 oracle.

Tolerances, from the arithmetic: u bounds the root mean square of a rounding's
relative error (2^-9 bfloat16, 2^-12 float16; 2^-24 float32).  An output is rounded once (u), and sums products
of probabilities rounded once (u, relative to a sum of terms of either sign,
whose 2-norm over random data is that of the result): 2 u, twice that allowed.
A gradient has one more rounded factor (dS, or o within D): 3 u, twice that
allowed.  In float32 nothing is rounded short; sums of up to some hundred terms and
exponentials of arguments up to 2^4 give a few times 2^4 u = 1e-6, and ten times
that is allowed.  Single values may be off by 8 times as much of the output's
root mean square or their own size, whichever is larger.
"""

import numpy as np
import pytest
import torch

from deepfold import _native as nat
from deepfold.model.kernels.flash_window_attn import flash_window_attn, window_attn_decode
from deepfold.model.position_encoding import RelativeBuckets, relative_position_bias
from oracle import window_attn_oracle as orc

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF16: 2.0 ** -9, F16: 2.0 ** -12}
BUCKETS = {"log": RelativeBuckets.log(32, 128, False), "log2": RelativeBuckets.log(32, 128, True),
           "clip": RelativeBuckets.clip(7), "far": RelativeBuckets.log(24, 700, True), "one": RelativeBuckets([0])}


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, dtype, rounds, what=""):
    got = f64(got)
    assert got.shape == want.shape, what
    assert np.isfinite(got).all(), what
    tol = 1e-5 if dtype == F32 else 2 * rounds * ROUND[dtype]
    norm = np.linalg.norm(want)
    rms = norm / max(1, want.size) ** 0.5
    assert np.linalg.norm(got - want) <= tol * norm + 1e-30, (what, np.linalg.norm(got - want) / (norm + 1e-300), tol)
    if want.size:
        assert (np.abs(got - want) <= 8 * tol * np.maximum(rms, np.abs(want)) + 1e-30).all(), what


def inputs(B, H, H_kv, n_q, n_k, d, dtype, seed=0, layout="bhnd", nb=None):
    g = torch.Generator().manual_seed(seed)

    def heads(h, n):
        if layout == "bnhd":
            return torch.randn(B, n, h, d, generator=g).to(dtype).cuda().transpose(1, 2)
        if layout == "packed":   # q, k and v as slices of one projection: rows one element off 16 bytes
            return torch.randn(B, n, h, d + 3, generator=g).to(dtype).cuda()[..., 1:d + 1].transpose(1, 2)
        return torch.randn(B, h, n, d, generator=g).to(dtype).cuda()
    x = dict(q=heads(H, n_q), k=heads(H_kv, n_k), v=heads(H_kv, n_k), d_o=heads(H, n_q))
    x["w"] = None if nb is None else (0.5 * torch.randn(H, nb, generator=g)).to(dtype).cuda()
    return x


def prefix_mask(lengths, n_k):
    return (torch.arange(n_k)[None] < torch.tensor(lengths)[:, None]).cuda()


def check(x, dtype, buckets=None, mask=None, grad=True, **kw):
    table = None if buckets is None else buckets.table
    w = x["w"] if buckets is not None else None
    want = orc.window_attn(f64(x["q"]), f64(x["k"]), f64(x["v"]), weight=None if w is None else f64(w), table=table,
                           mask=None if mask is None else f64(mask != 0), d_o=f64(x["d_o"]) if grad else None, **kw)
    leaves = [t.detach().requires_grad_(grad) for t in (x["q"], x["k"], x["v"])]
    wl = None if w is None else w.detach().requires_grad_(grad)
    o = flash_window_attn(*leaves, pos_weight=wl, buckets=buckets, mask=mask, **kw)
    assert o.dtype == dtype
    if not grad:
        close(o, want, dtype, 2, "o")
        return o
    close(o, want[0], dtype, 2, "o")
    got = torch.autograd.grad(o, leaves + ([] if wl is None else [wl]), x["d_o"])
    for name, a, b in zip(("d_q", "d_k", "d_v", "d_w"), got, want[1:]):
        assert a.dtype == dtype
        close(a, b, dtype, 3, name)
    return o, got


SHAPES = [  # B, H, H_kv, n_q, n_k, d, layout
    (1, 1, 1, 1, 1, 8, "bhnd"),
    (2, 4, 2, 17, 17, 32, "bnhd"),
    (1, 6, 2, 130, 130, 64, "bhnd"),
    (2, 2, 1, 5, 257, 40, "bnhd"),
    (1, 3, 3, 128, 384, 24, "bhnd"),
    (1, 2, 2, 300, 300, 33, "packed"),
    (1, 2, 1, 129, 64, 16, "bnhd"),    # more queries than keys: the first see nothing (causal)
]
WINDOWS = [  # causal, window, sinks, buckets
    (True, None, 0, "log"),
    (True, 16, 4, "log"),
    (True, 1, 0, None),
    (False, 40, 1, "log2"),
    (False, None, 0, "clip"),
    (True, 100, 70, "far"),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("causal,window,sinks,kind", WINDOWS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, causal, window, sinks, kind, dtype):
    B, H, H_kv, n_q, n_k, d, layout = shape
    buckets = BUCKETS[kind] if kind else None
    x = inputs(B, H, H_kv, n_q, n_k, d, dtype, 1, layout, buckets.num_buckets if buckets else None)
    # a query that sees one key has a gradient of exactly 0, which no relative tolerance measures
    one_key = window == 1 or n_k == 1
    check(x, dtype, buckets, causal=causal, window=window, sinks=sinks, grad=not one_key)


@pytest.mark.parametrize("causal,window,sinks,n_q,n_k,q_start,H,H_kv", [
    (True, 16, 4, 1537, 1537, None, 2, 1),     # many queries beyond the window see the sinks only
    (False, 30, 3, 1400, 1400, None, 1, 1),
    (True, 9, 200, 1700, 1700, None, 1, 1),    # sinks over two key tiles
    (True, 10, 3, 1600, 64, 0, 2, 2),          # few keys, queries far beyond them
    (False, 12, 2, 1300, 1500, 900, 1, 1)])
def test_gradients_of_sinks_that_many_queries_see(causal, window, sinks, n_q, n_k, q_start, H, H_kv):
    x = inputs(1, H, H_kv, n_q, n_k, 32, BF16, 16, nb=32)
    mask = torch.ones(1, n_k, device="cuda", dtype=torch.bool)
    mask[0, 1] = False
    check(x, BF16, BUCKETS["log2"], mask, causal=causal, window=window, sinks=sinks, q_start=q_start)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks_with_holes_empty_rows_and_nan_in_the_padding(dtype):
    n = 200
    mask = prefix_mask([200, 0, 70], n)
    mask[0, 30:150] = False   # with a window of 20, queries 50..130 see no key, in either direction
    mask[2, ::3] = False
    x = inputs(3, 2, 1, n, n, 32, dtype, 2, nb=32)
    hidden = ~mask[:, None, :, None]
    x["k"] = x["k"].masked_fill(hidden, float("nan"))
    x["v"] = x["v"].masked_fill(hidden, float("inf"))
    for causal in (True, False):
        o, grads = check(x, dtype, BUCKETS["log2"], mask, causal=causal, window=20, sinks=0)
        assert (o[0, :, 50:130] == 0).all() and (o[1] == 0).all()
        assert (grads[0][0, :, 50:130] == 0).all() and (grads[1][1] == 0).all()
        assert all(torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("mask_type", [torch.bool, torch.uint8, torch.float32, torch.int64])
def test_mask_types(mask_type):
    x = inputs(2, 2, 2, 40, 40, 16, F16, 3)
    mask = prefix_mask([40, 11], 40)
    want = flash_window_attn(x["q"], x["k"], x["v"], mask=mask)
    assert torch.equal(flash_window_attn(x["q"], x["k"], x["v"], mask=mask.to(mask_type)), want)


@pytest.mark.parametrize("q_start", [-30, 0, 7, 200, 5000])
def test_query_positions(q_start):
    x = inputs(1, 2, 2, 70, 150, 32, F32, 4, nb=32)
    for causal in (True, False):
        # from 200 on only the two sinks are seen, both in the last bucket: d_w is exactly 0, as with one key
        check(x, F32, BUCKETS["log2"], causal=causal, window=33, sinks=2, q_start=q_start, grad=q_start < 200)


def test_a_table_of_one_bucket_changes_nothing_but_the_gradient_of_a_constant():
    x = inputs(1, 2, 2, 50, 50, 16, F32, 5, nb=1)
    with_bias = flash_window_attn(x["q"], x["k"], x["v"], pos_weight=x["w"], buckets=BUCKETS["one"])
    close(with_bias, f64(flash_window_attn(x["q"], x["k"], x["v"])), F32, 2)


def test_bias_of_minus_infinity_hides_a_bucket():
    x = inputs(1, 2, 2, 90, 90, 32, F32, 6, nb=15)
    x["w"][:, 7] = float("-inf")  # clip(7): the bucket of delta = 0
    check(x, F32, BUCKETS["clip"], causal=True, window=20, sinks=0, grad=False)


def test_scale_and_unbatched_and_cpu():
    x = inputs(1, 2, 2, 33, 33, 16, F32, 7)
    check(x, F32, scale=1.7)
    q, k, v = x["q"][0], x["k"][0], x["v"][0]
    want = flash_window_attn(x["q"], x["k"], x["v"], window=9)
    assert torch.equal(flash_window_attn(q, k, v, window=9), want[0])
    assert torch.equal(flash_window_attn(q.cpu(), k.cpu(), v.cpu(), window=9), want[0].cpu())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_operands_and_gradients(dtype):
    """Expanded (stride 0) key heads and an expanded upstream gradient."""
    x = inputs(2, 4, 1, 66, 66, 32, dtype, 8)
    q = x["q"].requires_grad_()
    k1, v1 = x["k"].requires_grad_(), x["v"].requires_grad_()
    a = torch.autograd.grad(flash_window_attn(q, k1, v1, window=30).float().sum(), [q, k1, v1])
    b = torch.autograd.grad(flash_window_attn(q, k1.expand(2, 4, 66, 32), v1.expand(2, 4, 66, 32), window=30)
                            .float().sum(), [q, k1, v1])
    ones = torch.ones_like(x["d_o"])
    want = orc.window_attn(f64(q), f64(k1), f64(v1), window=30, d_o=f64(ones))
    assert torch.equal(a[0], b[0])
    close(a[0], want[1], dtype, 3)
    close(a[2], want[3], dtype, 3)
    for u, w in zip(b[1:], want[2:4]):
        close(u, w, dtype, 4)  # autograd adds the heads' rounded gradients


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_matches_differences(dtype):
    """The kernels' gradients against central differences of the float64 oracle along a random direction."""
    x = inputs(1, 2, 1, 140, 140, 32, dtype, 9, nb=32)
    kw = dict(window=50, sinks=3, causal=True)
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "w")]
    o = flash_window_attn(*leaves[:3], pos_weight=leaves[3], buckets=BUCKETS["log"], **kw)
    grads = torch.autograd.grad(o, leaves, x["d_o"])
    base = [f64(t) for t in leaves]
    rng = np.random.default_rng(0)
    for i, g in enumerate(grads):
        step = rng.normal(size=base[i].shape)

        def f(t):
            y = [b + t * step if k == i else b for k, b in enumerate(base)]
            return float((orc.window_attn(*y[:3], weight=y[3], table=BUCKETS["log"].table, **kw) * f64(x["d_o"])).sum())
        want = (f(1e-5) - f(-1e-5)) / 2e-5
        # a sum of g.size products of independent signs: its error is that of g's 2-norm times |step|'s rms of 1
        tol = (1e-5 if dtype == F32 else 6 * ROUND[dtype]) * float(np.linalg.norm(f64(g))) * 4 + 1e-6
        assert abs(float((f64(g) * step).sum()) - want) <= tol


def test_results_repeat_bit_for_bit_and_on_another_stream():
    x = inputs(2, 4, 2, 300, 300, 64, BF16, 10, nb=32)

    def step():
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "w")]
        o = flash_window_attn(*leaves[:3], window=100, sinks=4, pos_weight=leaves[3], buckets=BUCKETS["log"])
        return (o.detach(), *torch.autograd.grad(o, leaves, x["d_o"]))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_first_cuda_work_of_a_host_thread():
    """A thread that has made no CUDA call yet, its tensors from the allocator's cache: the tensor maps are
    encoded by the driver, which needs the thread's context bound first."""
    import threading
    x = inputs(1, 2, 2, 200, 200, 32, BF16, 15)
    want = flash_window_attn(x["q"], x["k"], x["v"], window=50)
    spare = [torch.empty_like(want) for _ in range(8)]
    del spare
    torch.cuda.synchronize()
    got = []
    t = threading.Thread(target=lambda: got.append(nat.ext().window_attn(x["q"], x["k"], x["v"], None, None, None, 0,
                                                                         50, 0, True, 0, 32 ** -0.5)))
    t.start()
    t.join()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_empty_sizes():
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=BF16)  # noqa: E731
    assert flash_window_attn(z(0, 2, 4, 16), z(0, 2, 4, 16), z(0, 2, 4, 16)).shape == (0, 2, 4, 16)
    assert flash_window_attn(z(1, 2, 0, 16), z(1, 2, 4, 16), z(1, 2, 4, 16)).shape == (1, 2, 0, 16)
    q = torch.ones(1, 2, 5, 16, device="cuda", dtype=BF16, requires_grad=True)
    k = z(1, 2, 0, 16).requires_grad_()
    o = flash_window_attn(q, k, k)
    assert (o == 0).all()
    d_q, d_k = torch.autograd.grad(o.sum(), [q, k])
    assert (d_q == 0).all() and d_k.shape == k.shape
    q, k = z(1, 2, 0, 16).requires_grad_(), torch.ones(1, 2, 5, 16, device="cuda", dtype=BF16, requires_grad=True)
    (d_k,) = torch.autograd.grad(flash_window_attn(q, k, k).sum(), [k])
    assert (d_k == 0).all()


# ---------------------------------------------------------------- one token over a cache
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,H,H_kv,n,d,layout,window,sinks,kind", [
    (1, 1, 1, 1, 8, "bhnd", None, 0, None),
    (3, 4, 2, 9, 32, "bnhd", 4, 1, "log"),
    (5, 16, 4, 700, 64, "bnhd", 128, 4, "log"),
    (4, 6, 2, 1000, 40, "bhnd", None, 0, "far"),
    (2, 24, 1, 2100, 64, "bhnd", 2000, 3, "log"),   # 24 query heads share one key head
    (3, 2, 2, 333, 33, "packed", 50, 60, "clip"),
])
def test_decode(B, H, H_kv, n, d, layout, window, sinks, kind, dtype):
    buckets = BUCKETS[kind] if kind else None
    x = inputs(B, H, H_kv, 1, n, d, dtype, 11, layout, buckets.num_buckets if buckets else None)
    lengths = [n - (n * b) // max(1, B - 1) for b in range(B)]  # from full to empty
    k, v = x["k"].clone(), x["v"].clone()
    for b, L in enumerate(lengths):  # rows that were never written
        k[b, :, L:] = float("nan")
        v[b, :, L:] = float("nan")
    if layout == "packed":
        pad = torch.empty(B, n, H_kv, d + 3, device="cuda", dtype=dtype)
        pad[..., 1:d + 1] = k.transpose(1, 2)
        k = pad[..., 1:d + 1].transpose(1, 2)
    q = x["q"][:, :, 0]
    got = window_attn_decode(q, k, v, torch.tensor(lengths, device="cuda"), window, sinks,
                             pos_weight=x["w"], buckets=buckets)
    assert got.dtype == dtype and got.shape == (B, H, d)
    for b, L in enumerate(lengths):
        if L == 0:
            assert (got[b] == 0).all()
            continue
        want = orc.window_attn(f64(x["q"][b:b + 1]), f64(x["k"][b:b + 1, :, :L]), f64(x["v"][b:b + 1, :, :L]),
                               window=window, sinks=sinks, weight=None if buckets is None else f64(x["w"]),
                               table=None if buckets is None else buckets.table)
        close(got[b:b + 1, :, None], want, dtype, 2)


def test_decode_agrees_with_the_last_row_of_the_forward_and_clamps_lengths():
    x = inputs(2, 8, 2, 300, 300, 64, BF16, 12, nb=32)
    kw = dict(window=90, sinks=4, pos_weight=x["w"], buckets=BUCKETS["log"])
    full = flash_window_attn(x["q"], x["k"], x["v"], **kw)[:, :, -1]
    q = x["q"][:, :, -1]
    one = window_attn_decode(q, x["k"], x["v"], torch.tensor([300, 300], device="cuda", dtype=torch.int32), **kw)
    close(one, f64(full), BF16, 4)  # two results, each rounded
    beyond = window_attn_decode(q, x["k"], x["v"], torch.tensor([9999, -3], device="cuda"), **kw)
    assert torch.equal(beyond[0], one[0]) and (beyond[1] == 0).all()


# ---------------------------------------------------------------- the dense bias
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("H,n_q,n_k,q_start,kind", [
    (1, 1, 1, 0, "log2"), (3, 5, 700, None, "log"), (2, 384, 384, 0, "clip"), (2, 129, 1001, -40, "far"),
    (4, 1000, 77, None, "log2"), (2, 40, 40, 3, "one"), (1, 33, 2050, 5000, "log")])
def test_dense_bias_and_its_gradient(H, n_q, n_k, q_start, kind, dtype):
    b = BUCKETS[kind]
    g = torch.Generator().manual_seed(13)
    w = torch.randn(H, b.num_buckets, generator=g).to(dtype).cuda().requires_grad_()
    up = torch.randn(H, n_q, n_k, generator=g).to(dtype).cuda()
    start = n_k - n_q if q_start is None else q_start
    want, buckets = orc.bias_matrix(f64(w), b.table, n_q, n_k, start)
    got = relative_position_bias(w, b, n_q, n_k, q_start)
    assert got.dtype == dtype and np.array_equal(f64(got), want)  # entries are copied: no rounding
    assert np.array_equal(f64(relative_position_bias(w.detach(), b, n_q, n_k, q_start)), want)
    (dw,) = torch.autograd.grad(got, [w], up)
    close(dw, orc.bias_grad(f64(up), buckets, b.num_buckets), dtype, 2)


def test_dense_bias_odd_views_and_empty_sizes():
    b = BUCKETS["log2"]
    w = torch.randn(3, 40, device="cuda", dtype=BF16)[:, 5:37].requires_grad_()  # rows 2 bytes off
    up = torch.randn(3, 130, 71, device="cuda", dtype=BF16)
    got = relative_position_bias(w, b, 71, 130)
    (dw,) = torch.autograd.grad(got, [w], up.transpose(1, 2))
    want, buckets = orc.bias_matrix(f64(w), b.table, 71, 130, 59)
    assert np.array_equal(f64(got), want)
    close(dw, orc.bias_grad(f64(up.transpose(1, 2)), buckets, 32), BF16, 2)
    (dw,) = torch.autograd.grad(relative_position_bias(w, b, 71, 130).sum(), [w])  # an expanded gradient
    close(dw, orc.bias_grad(np.ones((3, 71, 130)), buckets, 32), BF16, 2)
    assert relative_position_bias(w, b, 0, 9).shape == (3, 0, 9)
    (dw,) = torch.autograd.grad(relative_position_bias(w, b, 0, 9).sum(), [w])
    assert (dw == 0).all()


# ---------------------------------------------------------------- refusals
def test_refusals():
    x = inputs(1, 4, 2, 8, 8, 16, BF16, 14, nb=32)
    q, k, v, w = x["q"], x["k"], x["v"], x["w"]
    b = BUCKETS["log"]
    one = torch.ones(1, device="cuda", dtype=torch.int32)
    for kw in (dict(window=0), dict(sinks=-1), dict(scale=float("inf")), dict(pos_weight=w), dict(buckets=b),
               dict(pos_weight=w[:, :31], buckets=b)):
        with pytest.raises(ValueError):
            flash_window_attn(q, k, v, **kw)
        with pytest.raises(ValueError):
            window_attn_decode(q[:, :, 0], k, v, one, **kw)
    with pytest.raises(TypeError):
        flash_window_attn(q, k, v, pos_weight=w, buckets=[0, 1, 2])
    for bad in ((q, k.float(), v), (q.double(), k.double(), v.double()), (q[:, :3], k, v), (q, k, v[:, :, :7]),
                (q, k.cpu(), v), (q, k[..., :8], v[..., :8]), (q.repeat(1, 1, 1, 5), k.repeat(1, 1, 1, 5),
                                                            v.repeat(1, 1, 1, 5))):
        with pytest.raises(RuntimeError):
            flash_window_attn(*bad)
    for kw in (dict(mask=torch.ones(1, 7, device="cuda")), dict(mask=torch.ones(1, 8)),
               dict(pos_weight=w[:3], buckets=b), dict(pos_weight=w.double(), buckets=b), dict(q_start=1 << 40)):
        with pytest.raises(RuntimeError):
            flash_window_attn(q, k, v, **kw)
    for lengths in (one.float(), one.cpu(), torch.ones(2, device="cuda", dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            window_attn_decode(q[:, :, 0], k, v, lengths)
    with pytest.raises(NotImplementedError):
        window_attn_decode(q[:, :, 0].requires_grad_(), k, v, one)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_of_one_long_sequence(dtype):
    """Sixteen blocks join, and runs of keys end inside a tile."""
    x = inputs(1, 4, 2, 1, 5003, 64, dtype, 31, nb=32)
    got = window_attn_decode(x["q"][:, :, 0], x["k"], x["v"], torch.tensor([4990], device="cuda"),
                             pos_weight=x["w"], buckets=BUCKETS["log"])
    want = orc.window_attn(f64(x["q"]), f64(x["k"][:, :, :4990]), f64(x["v"][:, :, :4990]), weight=f64(x["w"]),
                           table=BUCKETS["log"].table)
    close(got[:, :, None], want, dtype, 2)


@pytest.mark.parametrize("causal,window,sinks,n,H,H_kv,d", [
    (True, None, 0, 900, 8, 1, 64),       # one key head: its tiles' steps are spread over many blocks
    (True, 150, 5, 1600, 8, 1, 40),       # with the sinks' far queries apart
    (False, 64, 140, 1100, 6, 1, 32),     # sinks over two key tiles, the keys' last tile ragged
])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_of_few_key_heads(causal, window, sinks, n, H, H_kv, d, dtype):
    x = inputs(1, H, H_kv, n, n, d, dtype, 37, "bnhd", 32)
    mask = prefix_mask([n - 130], n) if sinks == 5 else None
    _, first = check(x, dtype, BUCKETS["log"], mask, causal=causal, window=window, sinks=sinks)
    _, again = check(x, dtype, BUCKETS["log"], mask, causal=causal, window=window, sinks=sinks)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("causal,window,sinks,n_q,n_k,H,H_kv,d", [
    (True, None, 0, 5, 3001, 4, 2, 64),      # a few new tokens over a long past
    (True, None, 3, 1, 2048, 2, 2, 40),
    (True, 900, 4, 200, 4000, 3, 1, 32),
    (False, 700, 0, 130, 2100, 2, 2, 64),
    (True, None, 0, 1000, 1000, 1, 1, 64),   # the first tiles have fewer keys than there are blocks
])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_queries_over_many_keys(causal, window, sinks, n_q, n_k, H, H_kv, d, dtype):
    x = inputs(2, H, H_kv, n_q, n_k, d, dtype, 41, "bnhd", 32)
    mask = prefix_mask([n_k, n_k // 3], n_k)
    if n_q > 1:
        mask[1, :n_k // 4] = False
    check(x, dtype, BUCKETS["log"], mask, causal=causal, window=window, sinks=sinks)
    check(x, dtype, BUCKETS["log"], None, causal=causal, window=window, sinks=sinks, grad=False)


def test_few_queries_that_see_nothing():
    x = inputs(1, 2, 1, 40, 2048, 64, BF16, 43, nb=32)
    mask = torch.zeros(1, 2048, dtype=torch.bool, device="cuda")
    o, grads = check(x, BF16, BUCKETS["log"], mask, causal=True)
    assert (o == 0).all() and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_key_is_a_sink(dtype):
    """Sinks over all key tiles: their far queries outnumber the near ones everywhere."""
    n = 1900
    x = inputs(1, 2, 1, n, n, 32, dtype, 47, nb=32)
    check(x, dtype, BUCKETS["log"], causal=True, window=16, sinks=n)


def test_captured_in_a_graph():
    """A decoding step, and a forward with gradients, replayed on new inputs."""
    x = inputs(2, 4, 2, 260, 260, 64, BF16, 53, nb=32)
    kw = dict(window=100, sinks=4, buckets=BUCKETS["log"])
    q, k, v, w = (x[n].detach().clone().requires_grad_() for n in ("q", "k", "v", "w"))
    lengths = torch.tensor([260, 31], device="cuda", dtype=torch.int32)

    def work():
        with torch.no_grad():
            one = window_attn_decode(q[:, :, 0], k, v, lengths, pos_weight=w, **kw)
            few = flash_window_attn(q[:, :, :3], k, v, causal=False, pos_weight=w, **kw)
        o = flash_window_attn(q, k, v, pos_weight=w, **kw)
        return (one, few, o.detach(), *torch.autograd.grad(o, (q, k, v, w), x["d_o"]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    fresh = inputs(2, 4, 2, 260, 260, 64, BF16, 54, nb=32)
    with torch.no_grad():
        for t, n in ((q, "q"), (k, "k"), (v, "v"), (w, "w")):
            t.copy_(fresh[n])
        lengths.copy_(torch.tensor([7, 200]))
    graph.replay()
    got = [t.clone() for t in got]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, work()))
    del graph
