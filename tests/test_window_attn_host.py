"""Local attention without a GPU: the bucket tables, the oracle's gradients
against differences, the C entry points' and the Python surface's refusals."""

import ctypes
import math

import numpy as np
import pytest
import torch

from deepfold import _native as nat
from deepfold.model.kernels.flash_window_attn import flash_window_attn, window_attn_decode
from deepfold.model.position_encoding import RelativeBuckets, relative_position_bias
from oracle import window_attn_oracle as orc


def log_rule(delta, nb, D, both):
    """The bucket rule with real logarithms (1e-9 of slack at a step's edge)."""
    side = nb // 2 if both else nb
    first = nb - side if both and delta < 0 else 0
    n = abs(delta) if both else max(delta, 0)
    near = side // 2
    if n < near:
        return first + n
    step = math.floor(math.log(min(n, D) / near) / math.log(D / near) * (side - near) + 1e-9)
    return first + min(near + step, side - 1)


@pytest.mark.parametrize("nb,D,both", [(32, 128, True), (32, 128, False), (16, 40, False), (24, 600, True),
                                       (4, 1024, True), (7, 9, False)])
def test_log_buckets_follow_the_rule(nb, D, both):
    b = RelativeBuckets.log(nb, D, both)
    assert b.max_distance == D and b.num_buckets == nb
    assert list(b.table) == [log_rule(x, nb, D, both) for x in range(-D, D + 1)]


def test_clip_buckets_are_compute_bins_rule_within_a_chain():
    b = RelativeBuckets.clip(32)
    assert b.num_buckets == 65
    assert list(b.table) == [min(max(x, -32), 32) + 32 for x in range(-32, 33)]


@pytest.mark.parametrize("table,nb", [([0, 1], None), ([0] * (2 * 1024 + 3), None), ([0, 3, 1], 3), ([0, -1, 1], 3)])
def test_bucket_tables_that_are_refused(table, nb):
    with pytest.raises(ValueError):
        RelativeBuckets(table, nb)


@pytest.mark.parametrize("kw", [dict(num_buckets=3), dict(num_buckets=32, max_distance=8),
                                dict(num_buckets=1, bidirectional=False)])
def test_log_bucket_sizes_that_are_refused(kw):
    with pytest.raises(ValueError):
        RelativeBuckets.log(**kw)


@pytest.mark.parametrize("causal,window,sinks", [(True, None, 0), (True, 3, 2), (False, 4, 1)])
def test_oracle_gradient_matches_differences(causal, window, sinks):
    rng = np.random.default_rng(5)
    B, H, H_kv, n_q, n_k, d = 2, 4, 2, 6, 9, 3
    x = {"q": rng.normal(size=(B, H, n_q, d)), "k": rng.normal(size=(B, H_kv, n_k, d)),
         "v": rng.normal(size=(B, H_kv, n_k, d)), "weight": rng.normal(size=(H, 5))}
    mask = np.ones((B, n_k))
    mask[1, 4:] = 0
    d_o = rng.normal(size=(B, H, n_q, d))
    kw = dict(causal=causal, window=window, sinks=sinks, table=[0, 1, 2, 3, 4], mask=mask)
    grads = dict(zip(("q", "k", "v", "weight"), orc.window_attn(**x, **kw, d_o=d_o)[1:]))
    for name in x:
        step = rng.normal(size=x[name].shape)
        f = lambda t: float((orc.window_attn(**{**x, name: x[name] + t * step}, **kw) * d_o).sum())  # noqa: E731
        h = 1e-5  # central differences: error h^2 / 6 times a third derivative of order 10 to 100, and 1e-16 / h
        assert abs((f(h) - f(-h)) / (2 * h) - float((grads[name] * step).sum())) < 1e-7, name


def test_struct_sizes_match_header_layout():
    assert ctypes.sizeof(nat.DfsRelBias) == 32
    assert ctypes.sizeof(nat.DfsAttnProblem) == 48
    assert ctypes.sizeof(nat.DfsStrided) == 32
    assert ctypes.sizeof(nat.DfsAttnArgs) == 8 * 32 + 32 + 5 * 8


def attn(**kw):
    base = dict(B=2, H=4, H_kv=2, n_q=8, n_k=8, d=32, dtype=nat.DFS_BF16, causal=1, window=4, sinks=1, q_start=0,
                scale=0.2)
    return nat.DfsAttnProblem(**{**base, **kw})


E, U = nat.DFS_ERR_INVALID_ARGUMENT, nat.DFS_ERR_UNSUPPORTED
BAD_PROBLEMS = [(dict(B=-1), E), (dict(H_kv=3), E), (dict(H_kv=0), E), (dict(n_q=-2), E), (dict(d=0), E),
                (dict(dtype=7), E), (dict(window=-1), E), (dict(sinks=-1), E), (dict(scale=float("nan")), E),
                (dict(d=65), U), (dict(n_k=(1 << 28) + 1), U), (dict(q_start=1 << 30), U)]


@pytest.mark.parametrize("kw,code", BAD_PROBLEMS)
def test_entry_points_refuse_bad_problems(kw, code):
    lib, a = nat.lib(), nat.DfsAttnArgs()
    p = attn(**kw)
    assert lib.dfs_window_attn_fwd(p, a, None) == code
    assert lib.dfs_window_attn_bwd(p, a, None, 0, None) == code
    assert lib.dfs_window_attn_bwd_work(p, a.bias) == 0
    if p.n_q > 0:
        p.n_q = 1
        assert lib.dfs_window_attn_decode(p, a, None, None) == code


def test_entry_points_refuse_missing_buffers_and_bad_tables():
    lib = nat.lib()
    p, none = attn(), nat.DfsAttnArgs()
    for rc in (lib.dfs_window_attn_fwd(p, none, None), lib.dfs_window_attn_fwd(p, None, None),
               lib.dfs_window_attn_fwd(None, none, None), lib.dfs_window_attn_bwd(p, none, None, 0, None),
               lib.dfs_window_attn_decode(p, none, None, None), lib.dfs_window_attn_decode(attn(n_q=1), none, None, None)):
        assert rc == E
    s = nat.DfsStrided(ptr=16)
    full = dict(q=s, k=s, v=s, o=s, lse=16, d_o=s, d_q=s, d_k=s, d_v=s)
    assert lib.dfs_window_attn_bwd(p, nat.DfsAttnArgs(**full, d_weight=16), 16, 1 << 30, None) == E  # no weight
    assert lib.dfs_window_attn_bwd(p, nat.DfsAttnArgs(**full), 16, 0, None) == nat.DFS_ERR_WORKSPACE
    for bad in (dict(lut=None), dict(num_buckets=0), dict(max_distance=1025), dict(max_distance=-1), dict(dtype=5)):
        b = nat.DfsRelBias(**{**dict(weight=16, lut=16, num_buckets=3, max_distance=1, dtype=0), **bad})
        assert lib.dfs_window_attn_fwd(p, nat.DfsAttnArgs(**full, bias=b), None) == E
        assert lib.dfs_relbias_fwd(1, 4, 4, 0, b, 16, None) == E
        assert lib.dfs_relbias_bwd(1, 4, 4, 0, b, 16, 16, 16, 1 << 20, None) == E
        assert lib.dfs_relbias_bwd_work(1, 4, 4, b) == 0
    b = nat.DfsRelBias(weight=16, lut=16, num_buckets=3, max_distance=1, dtype=0)
    assert lib.dfs_relbias_fwd(1, -4, 4, 0, b, 16, None) == E
    assert lib.dfs_relbias_fwd(1, 4, 4, 0, b, None, None) == E
    assert lib.dfs_relbias_bwd(1, 4, 4, 0, b, None, 16, 16, 1 << 20, None) == E
    assert lib.dfs_relbias_bwd(1, 4, 4, 0, b, 16, 16, 16, 0, None) == nat.DFS_ERR_WORKSPACE


def test_empty_problems_are_done_without_a_device():
    lib, none = nat.lib(), nat.DfsAttnArgs()
    for kw in (dict(B=0), dict(H=0, H_kv=0), dict(n_q=0)):
        assert lib.dfs_window_attn_fwd(attn(**kw), none, None) == nat.DFS_OK
    assert lib.dfs_window_attn_bwd(attn(B=0), none, None, 0, None) == nat.DFS_OK
    b = nat.DfsRelBias(weight=16, lut=16, num_buckets=3, max_distance=1, dtype=0)
    assert lib.dfs_relbias_fwd(2, 0, 5, 0, b, None, None) == nat.DFS_OK


def test_python_surface_refuses_on_the_host():
    x = torch.zeros(1, 2, 4, 8)
    if not torch.cuda.is_available():
        for call in (lambda: flash_window_attn(x, x, x), lambda: window_attn_decode(x[:, :, 0], x, x, torch.ones(1)),
                     lambda: relative_position_bias(torch.zeros(2, 65), RelativeBuckets.clip(), 4, 4)):
            with pytest.raises(RuntimeError, match="CUDA device"):
                call()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nat.ext().window_attn(x, x, x, None, None, None, 0, 0, 0, True, 0, 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nat.ext().relative_position_bias(torch.zeros(2, 3), torch.zeros(3, dtype=torch.int32), 1, 4, 4, 0)
    with pytest.raises(ValueError, match="number of buckets"):
        relative_position_bias(torch.zeros(2, 64), RelativeBuckets.clip(), 4, 4)
    with pytest.raises(TypeError):
        relative_position_bias(torch.zeros(2, 64), [0, 1, 2], 4, 4)
    with pytest.raises(ValueError):
        relative_position_bias(torch.zeros(2, 65), RelativeBuckets.clip(), -1, 4)


@pytest.mark.parametrize("n,window,sinks,H,H_kv,B", [
    (65536, 16, 65536, 16, 16, 1), (65536, 16, 4, 16, 2, 1), (65536, 0, 0, 16, 16, 2), (2048, 0, 0, 32, 1, 1),
    (20000, 1, 300, 8, 8, 3)])
def test_backward_workspace_stays_in_proportion(n, window, sinks, H, H_kv, B):
    """At most a float a query and, where blocks share key tiles, 1 KB a key and block (sinks: a block more at most
    per key tile; few key heads: up to two blocks an SM)."""
    p = attn(B=B, H=H, H_kv=H_kv, n_q=n, n_k=n, d=64, window=window, sinks=sinks)
    work = nat.lib().dfs_window_attn_bwd_work(p, None)
    sink_rows = min(sinks, 128) * (n // 128 + min(sinks, n) // 128 + 2) * B * H_kv
    assert 4 * B * H * n <= work <= 4 * B * H * n + 512 * sink_rows + 2 * 148 * 128 * 512 + 1024
