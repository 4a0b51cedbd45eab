"""Local attention and its position bias at the edges of what a call may be given: empty problems, values that are
not finite or very large, derivatives that it does not have, other threads.  Tolerances as in test_gpu_window_attn.py
unless a test derives its own."""

import threading
import time

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from deepfold import _native as nat
from deepfold.model.kernels.flash_window_attn import check_status, flash_window_attn, window_attn_decode
from deepfold.model.kernels import sinkhorn_kernel
from deepfold.model.position_encoding import RelativeBuckets, relative_position_bias
from oracle import window_attn_oracle as orc

from test_gpu_window_attn import BF16, BUCKETS, F16, F32, ROUND, check, f64, inputs

pytestmark = pytest.mark.gpu


def poison(*shape, dtype=F32):
    """Leaves blocks of NaN of this size in the allocator's cache, for the call's outputs to be made in."""
    spare = [torch.full(shape, float("nan"), device="cuda", dtype=dtype) for _ in range(8)]
    torch.cuda.synchronize()
    del spare


def test_bias_gradient_of_an_empty_batch_is_zero():
    w = torch.ones(3, 32, device="cuda", requires_grad=True)
    q = torch.zeros(0, 3, 5, 16, device="cuda", dtype=BF16)
    poison(3, 32)
    (d_w,) = torch.autograd.grad(flash_window_attn(q, q, q, pos_weight=w, buckets=BUCKETS["log"]).sum(), [w])
    assert (d_w == 0).all()


@pytest.mark.parametrize("dtype,code", [(F32, nat.DFS_F32), (BF16, nat.DFS_BF16)])
def test_c_entry_writes_the_bias_gradient_of_an_empty_batch(dtype, code):
    lut = torch.zeros(3, device="cuda", dtype=torch.int32)
    w = torch.ones(2, 5, device="cuda", dtype=dtype)
    d_w = torch.full_like(w, float("nan"))
    p = nat.DfsAttnProblem(B=0, H=2, H_kv=1, n_q=4, n_k=4, d=16, dtype=code, causal=1, scale=1.0)
    bias = nat.DfsRelBias(weight=w.data_ptr(), lut=lut.data_ptr(), num_buckets=5, max_distance=1, dtype=code)
    a = nat.DfsAttnArgs(bias=bias, d_weight=d_w.data_ptr())
    assert nat.lib().dfs_window_attn_bwd(p, a, None, 0, nat.stream_ptr(w.device)) == nat.DFS_OK
    assert (d_w == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_key_gradients_without_query_heads_are_zero(dtype):
    q = torch.zeros(2, 0, 5, 16, device="cuda", dtype=dtype, requires_grad=True)
    k, v = (torch.ones(2, 3, 70, 16, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
    w = torch.ones(0, 32, device="cuda", requires_grad=True)
    for kw, leaves in ((dict(), [k, v]), (dict(pos_weight=w, buckets=BUCKETS["log"], window=4, sinks=1), [k, v, w])):
        o = flash_window_attn(q, k, v, **kw)
        poison(2, 3, 70, 16, dtype=dtype)
        grads = torch.autograd.grad(o.sum(), leaves)
        assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, leaves))


def plain(q, k, v, w, table):
    """Causal attention with a bias as float64 softmax: what is not finite spreads as the formula has it."""
    q, k, v, w = (t.detach().double().cpu() for t in (q, k, v, w))
    G, (n_q, n_k), D = q.shape[1] // k.shape[1], (q.shape[2], k.shape[2]), len(table) // 2
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    delta = (torch.arange(n_q) + n_k - n_q)[:, None] - torch.arange(n_k)[None]
    bias = w[:, torch.tensor(table)[delta.clamp(-D, D) + D]]
    s = (q @ k.mT * q.shape[-1] ** -0.5 + bias).masked_fill(delta < 0, float("-inf"))
    p = torch.softmax(s, -1).masked_fill(delta < 0, 0.0)
    return (p @ v).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [40, 5003])  # one block, and sixteen that join
@pytest.mark.parametrize("what", ["q", "k", "v", "w", "logit"])
def test_what_is_not_finite_shows_in_the_token(what, n, dtype):
    """NaN in q, in a visible key, value or weight, or a logit of +inf: NaN where the formula has it, as the forward."""
    x = inputs(2, 4, 2, 1, n, 32, dtype, 61, nb=32)
    at = {"q": x["q"][0, 1, 0], "k": x["k"][0, 0, n - 2], "v": x["v"][0, 0, n - 2], "w": x["w"][1]}
    at.get(what, x["w"][1])[0] = float("inf") if what == "logit" else float("nan")
    kw = dict(pos_weight=x["w"], buckets=BUCKETS["log"])
    one = window_attn_decode(x["q"][:, :, 0], x["k"], x["v"], torch.tensor([n, n], device="cuda"), **kw)
    full = flash_window_attn(x["q"], x["k"], x["v"], **kw)[:, :, 0]
    want = plain(x["q"], x["k"], x["v"], x["w"], BUCKETS["log"].table)[:, :, 0]
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    assert torch.equal(torch.isnan(one), torch.isnan(want)) and torch.equal(torch.isnan(full), torch.isnan(want))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", ["k", "w"])
def test_gradients_of_a_row_that_is_not_finite(what, dtype):
    """A query whose softmax is NaN gives every key that it sees a NaN gradient, not that of a query that sees none."""
    x = inputs(1, 2, 1, 150, 150, 32, dtype, 67, nb=32)
    if what == "k":
        x["k"][0, 0, 60, 1] = float("nan")   # seen from query 60 on
    else:
        x["w"][:, 3] = float("inf")          # the bucket of delta = 3: every query from 3 on
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o = flash_window_attn(*leaves, pos_weight=x["w"], buckets=BUCKETS["log"])
    d_q, d_k, d_v = torch.autograd.grad(o, leaves, x["d_o"])
    first = 60 if what == "k" else 3
    assert torch.isnan(o[:, :, first:]).all() and torch.isfinite(o[:, :, :first]).all()
    assert torch.isnan(d_q[:, :, first:]).all()
    assert torch.isnan(d_k).all() and torch.isnan(d_v).all()  # the last query sees every key


def test_forward_mode_derivatives_are_refused():
    x = inputs(1, 2, 2, 20, 20, 16, F32, 71, nb=32)
    q, k, v, w, b = x["q"], x["k"], x["v"], x["w"], BUCKETS["log"]
    one = torch.tensor([20], device="cuda")
    with forward_ad.dual_level():
        d = {n: forward_ad.make_dual(x[n], torch.ones_like(x[n])) for n in ("q", "k", "v", "w")}
        for call in (lambda: flash_window_attn(d["q"], k, v), lambda: flash_window_attn(q, d["k"], v),
                     lambda: flash_window_attn(q, k, d["v"]),
                     lambda: flash_window_attn(q, k, v, pos_weight=d["w"], buckets=b),
                     lambda: window_attn_decode(d["q"][:, :, 0], k, v, one),
                     lambda: window_attn_decode(q[:, :, 0], k, v, one, pos_weight=d["w"], buckets=b),
                     lambda: relative_position_bias(d["w"], b, 4, 4)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_second_derivatives_are_refused():
    """Under create_graph the gradients are what they are without it; to differentiate them again raises."""
    x = inputs(1, 2, 1, 20, 20, 16, F32, 73, nb=32)
    q, k, v, w = leaves = [x[n].requires_grad_() for n in ("q", "k", "v", "w")]
    b = BUCKETS["log"]
    for out, of in ((flash_window_attn(q, k, v, pos_weight=w, buckets=b), leaves), (relative_position_bias(w, b, 9, 9), [w])):
        plain_grads = torch.autograd.grad(out.square().sum(), of, retain_graph=True)
        grads = torch.autograd.grad(out.square().sum(), of, create_graph=True)
        for t, g, want in zip(of, grads, plain_grads):
            assert g.requires_grad and not want.requires_grad and torch.equal(g, want)
            with pytest.raises(RuntimeError, match="once"):
                (t.sum() + g.square().sum()).backward(retain_graph=True)


def test_training_after_a_first_call_in_inference_mode():
    x = inputs(1, 2, 1, 20, 20, 16, F32, 79, nb=32)
    b = RelativeBuckets(BUCKETS["log"].table)
    with torch.inference_mode():
        first = flash_window_attn(x["q"], x["k"], x["v"], pos_weight=x["w"], buckets=b)
    w = x["w"].requires_grad_()
    o = flash_window_attn(x["q"], x["k"], x["v"], pos_weight=w, buckets=b)
    (o.sum() + relative_position_bias(w, b, 7, 7).sum()).backward()
    assert torch.equal(o.detach(), first) and torch.isfinite(w.grad).all()


@pytest.mark.parametrize("dtype,code", [(F32, nat.DFS_F32), (BF16, nat.DFS_BF16)])
def test_threads_with_tables_of_different_sizes(dtype, code):
    """The C entries from two host threads at once, one with the smallest table and one with the largest: neither
    thread's call takes the shared memory that the other's launch needs."""
    lib, failed = nat.lib(), []

    def worker(D, steps=2000):
        n, d, H = 64, 32, 2
        t = {name: torch.ones(1, H, n, d, device="cuda", dtype=dtype) for name in
             ("q", "k", "v", "o", "d_o", "d_q", "d_k", "d_v")}
        lse = torch.empty(1, H, n, device="cuda")
        w, d_w = (torch.ones(H, 4, device="cuda", dtype=dtype) for _ in range(2))
        lut = torch.zeros(2 * D + 1, dtype=torch.int32, device="cuda")
        length = torch.tensor([n], dtype=torch.int32, device="cuda")
        at = {name: nat.DfsStrided(ptr=x.data_ptr(), stride_b=H * n * d, stride_h=n * d, stride_n=d)
              for name, x in t.items()}
        bias = nat.DfsRelBias(weight=w.data_ptr(), lut=lut.data_ptr(), num_buckets=4, max_distance=D, dtype=code)
        a = nat.DfsAttnArgs(**at, lse=lse.data_ptr(), bias=bias, d_weight=d_w.data_ptr())
        p = nat.DfsAttnProblem(B=1, H=H, H_kv=H, n_q=n, n_k=n, d=d, dtype=code, causal=1, scale=0.2)
        one = nat.DfsAttnProblem(B=1, H=H, H_kv=H, n_q=1, n_k=n, d=d, dtype=code, causal=1, scale=0.2)
        size = lib.dfs_window_attn_bwd_work(p, bias)
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        for _ in range(steps):
            rc = (lib.dfs_window_attn_fwd(p, a, stream.cuda_stream),
                  lib.dfs_window_attn_bwd(p, a, work.data_ptr(), size, stream.cuda_stream),
                  lib.dfs_window_attn_decode(one, a, length.data_ptr(), stream.cuda_stream))
            if any(rc):
                failed.append((D, rc))
                break
        stream.synchronize()
    threads = [threading.Thread(target=worker, args=(D,)) for D in (0, 1024)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_lengths_beyond_32_bits_are_clamped():
    x = inputs(5, 2, 2, 1, 50, 16, F32, 83)
    lengths = torch.tensor([2 ** 32 + 5, 2 ** 40, -2 ** 40, 2 ** 31, -2 ** 31 - 7], device="cuda")
    got = window_attn_decode(x["q"][:, :, 0], x["k"], x["v"], lengths)
    want = window_attn_decode(x["q"][:, :, 0], x["k"], x["v"], torch.tensor([50, 50, 0, 50, 0], device="cuda"))
    assert torch.equal(got, want)


def test_a_device_error_is_reported_to_the_attention_that_met_it():
    """Not by the Sinkhorn operators' check, which neither raises for it nor takes it away; and once."""
    x = inputs(1, 2, 2, 20, 20, 16, F32, 89)
    q, k, v = x["q"], x["k"], x["v"]
    one = torch.tensor([20], device="cuda")
    want = flash_window_attn(q, k, v)
    torch.cuda.synchronize()
    for call in (check_status, lambda: check_status(wait=False), lambda: flash_window_attn(q, k, v),
                 lambda: window_attn_decode(q[:, :, 0], k, v, one)):
        nat.ext().window_attn_plant_status(nat.DFS_ERR_DEVICE_TIMEOUT)
        sinkhorn_kernel.check_status()
        with pytest.raises(RuntimeError, match="previous window attention call"):
            call()
        check_status()
        assert torch.equal(flash_window_attn(q, k, v), want)


LOWEST = [(F32, -1e9), (F32, torch.finfo(F32).min), (F32, 1e9), (BF16, -1e9), (BF16, torch.finfo(BF16).min),
          (F16, torch.finfo(F16).min)]


@pytest.mark.parametrize("dtype,low", LOWEST)
def test_rows_that_see_only_keys_of_one_very_large_bias(dtype, low):
    """A bias that all of a row's keys have changes nothing, whatever its size.  Logits and log-sums are held in steps
    of 2^-9 there: each p is off by 2^-10 of itself at most for either, beside the roundings of the type."""
    x = inputs(1, 2, 1, 150, 150, 32, dtype, 97, nb=32)
    x["w"][:] = low
    kw = dict(pos_weight=x["w"], buckets=BUCKETS["log"], window=70)
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o = flash_window_attn(*leaves, **kw)
    got = (o, *torch.autograd.grad(o, leaves, x["d_o"]),
           window_attn_decode(x["q"][:, :, -1], x["k"], x["v"], torch.tensor([150], device="cuda"), **kw))
    want = orc.window_attn(f64(x["q"]), f64(x["k"]), f64(x["v"]), window=70, d_o=f64(x["d_o"]))[:4]
    tol = 2 * 2.0 ** -10 + 2 * 3 * ROUND.get(dtype, 0.0) + 1e-5
    for a, b in zip(got, (*want, want[0][:, :, -1])):
        assert np.linalg.norm(f64(a) - b) <= tol * np.linalg.norm(b)


@pytest.mark.parametrize("dtype,low", LOWEST)
def test_a_very_low_bias_beside_others_hides(dtype, low):
    x = inputs(1, 2, 1, 150, 150, 32, dtype, 101, nb=32)
    x["w"][:, 9:] = -abs(low)   # a distance of 0 to 8 is seen by every query
    grads = []
    for w in (x["w"], torch.where(x["w"] == x["w"][0, 9], float("-inf"), x["w"])):
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v")]
        o = flash_window_attn(*leaves, pos_weight=w, buckets=BUCKETS["log"])
        one = window_attn_decode(x["q"][:, :, -1], x["k"], x["v"], torch.tensor([150], device="cuda"), pos_weight=w,
                                 buckets=BUCKETS["log"])
        grads.append((o, one, *torch.autograd.grad(o, leaves, x["d_o"])))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def run_out(which):
    """(seconds, status) of a block whose wait cannot succeed."""
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    start = time.monotonic()
    nat.check(nat.lib().dfs_selftest_wait(which, status.data_ptr(), nat.stream_ptr(status.device)), "dfs_selftest_wait")
    torch.cuda.synchronize()
    return time.monotonic() - start, int(status.item())


def test_a_wait_that_runs_out_ends_in_seconds():
    seconds, status = run_out(0)
    assert status == nat.DFS_ERR_DEVICE_TIMEOUT
    assert 1.0 < seconds < 10.0  # far above any wait of a kernel that works; bounded all the same


def test_copies_land_before_a_block_that_gave_up_ends():
    assert run_out(1)[1] == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("window,sinks,n_q,n_k,q_start", [
    (10, 148, 339, 339, None),    # the first queries' windows end tiles before the last sink
    (3, 700, 130, 900, 200),
    (1, 300, 70, 300, -5),
    (20, 64, 40, 400, -30),       # some queries stand before the first key
])
def test_sinks_ahead_of_the_window(window, sinks, n_q, n_k, q_start, dtype):
    """Without causality a query also sees the sinks that lie beyond its window's end."""
    x = inputs(2, 4, 2, n_q, n_k, 32, dtype, 103, nb=32)
    check(x, dtype, BUCKETS["log2"], causal=False, window=window, sinks=sinks, q_start=q_start)
