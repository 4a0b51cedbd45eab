"""Local attention's edges that need no GPU: what its calls refuse and keep on the host."""

import pytest
import torch
from torch.autograd import forward_ad

from deepfold import _native as nat
from deepfold.model.position_encoding import RelativeBuckets


def test_forward_mode_derivatives_are_refused():
    """Before anything else, with or without gradients: a tangent that is dropped reads as a derivative of 0."""
    x, w, lut = torch.ones(1, 2, 4, 8), torch.ones(2, 3), torch.zeros(3, dtype=torch.int32)
    ext = nat.ext()
    with forward_ad.dual_level():
        dual, dual_w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w))
        for call in (lambda: ext.window_attn(dual, x, x, None, None, None, 0, 0, 0, True, 0, 1.0),
                     lambda: ext.window_attn(x, x, x, None, dual_w, lut, 1, 0, 0, True, 0, 1.0),
                     lambda: ext.window_attn_decode(x[:, :, 0], x, dual, torch.ones(1), None, None, 0, 0, 0, 1.0),
                     lambda: ext.relative_position_bias(dual_w, lut, 1, 4, 4, 0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_a_table_first_used_in_inference_mode_serves_training():
    b = RelativeBuckets.log(16, 40)
    with torch.inference_mode():
        first = b.on(torch.device("cpu"))
        made = RelativeBuckets.clip(4, device="cpu").on(torch.device("cpu"))
    assert not first.is_inference() and not made.is_inference()
    assert b.on(torch.device("cpu")) is first and first.tolist() == list(b.table)


def test_the_entry_for_64_bit_lengths_refuses_as_the_other_does():
    lib, none = nat.lib(), nat.DfsAttnArgs()
    p = nat.DfsAttnProblem(B=2, H=4, H_kv=2, n_q=1, n_k=8, d=32, dtype=nat.DFS_BF16, causal=1, scale=0.2)
    for call in (lib.dfs_window_attn_decode, lib.dfs_window_attn_decode_i64):
        assert call(p, none, None, None) == call(p, None, None, None) == nat.DFS_ERR_INVALID_ARGUMENT
        p.B = 0
        assert call(p, none, None, None) == nat.DFS_OK
        p.B = 2


def test_the_wait_check_refuses_what_it_does_not_know():
    for which, status in ((-1, 16), (9, 16), (0, None)):
        assert nat.lib().dfs_selftest_wait(which, status, None) == nat.DFS_ERR_INVALID_ARGUMENT
