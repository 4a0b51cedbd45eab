"""Local softmax attention: a sliding window, a few first tokens that stay
visible (sinks), and a learned relative position bias by buckets.

* ``flash_window_attn``: the layer's forward, differentiable in Q, K, V and
  ``pos_weight`` (the N x N matrices are never built, forward or backward);
* ``window_attn_decode``: the same attention for the newest token of each
  sequence over a cache.

Neither is a drop-in for the reference's own softmax attention
(src/deepfold/model/kernels/flash_diffusion_attn.py, with its 68-bin bias;
flash_atom_attn.py, over a local window).  With delta = i + q_start - j, a key j
is visible to a query i when its ``mask`` entry is nonzero, it is not in the
future (``causal``: delta >= 0), and it is near (0 <= delta < window; without
``causal`` |delta| < window) or one of the first ``sinks`` keys.  A query that
sees no key gives zeros and gets zero gradients.  Keys hidden by ``mask`` are
never used, whatever they hold (padding may be NaN); keys hidden by the window
or by causality must be finite, as any real token's are.

Types: bfloat16 and float16 (tensor-core products, softmax statistics and all
sums in fp32; the probabilities and, in the backward, the logits' gradients are
rounded to the operands' type for the products that they enter, so an output is
about 1.3 and a gradient 1.5 times as far off as the exact one rounded once) and
float32 (fp32 products throughout).  With float16, upstream gradients much below
1e-4 meet the type's smallest values in those products: scale the loss.
Head dims 1 to 64; any strides with unit stride along d.  Head counts may differ
(H a multiple of H_kv: shared key heads, whose gradients are summed over the
group in a fixed order).  Results are bitwise reproducible.

The gradients are first ones in reverse mode: a second differentiation and
forward-mode derivatives raise.  A device error raises from the next attention call, or from ``check_status``.

CPU tensors are computed on the current CUDA device and the results returned on
the CPU; without a CUDA device the calls raise (there is no CPU path).
"""

from __future__ import annotations

import math

import torch

from deepfold import _native as nat
from deepfold.model.position_encoding import RelativeBuckets, check_buckets

__all__ = ["flash_window_attn", "window_attn_decode", "check_status"]


def check_status(wait: bool = True) -> None:
    """RuntimeError if an attention call made so far on the current device met a
    device error (a bounded wait of a kernel that gave up); without ``wait`` only
    if a call that has finished did.  The next attention call raises by itself;
    this makes the check immediate."""
    nat.ext().window_attn_check_status(bool(wait))


def _gpu(t):
    if not torch.cuda.is_available():
        raise RuntimeError("deepfold B200 attention runs on a CUDA device; none is available (no CPU path)")
    return t.to(torch.device("cuda", torch.cuda.current_device())) if isinstance(t, torch.Tensor) else t


def _options(d, window, sinks, scale, pos_weight, buckets, device):
    """Checked (window or 0, scale, bucket table, its distance)."""
    if window is not None and window < 1:
        raise ValueError("window must be at least 1 (None: no window)")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if (pos_weight is None) != (buckets is None):
        raise ValueError("pos_weight and buckets are given together")
    if pos_weight is None:
        return min(window or 0, 1 << 30), scale, None, 0
    check_buckets(pos_weight, buckets)
    return min(window or 0, 1 << 30), scale, buckets.on(device), buckets.max_distance


def flash_window_attn(Q, K, V, window: int | None = None, sinks: int = 0, causal: bool = True,
                      pos_weight=None, buckets: RelativeBuckets | None = None, mask=None,
                      q_start: int | None = None, scale: float | None = None):
    """Softmax attention over a sliding window and the first ``sinks`` keys.

    Q (B,H,n_q,d), K and V (B,H_kv,n_k,d); unbatched inputs drop B.  pos_weight
    (H, num_buckets) with ``buckets``: the learned bias (-inf hides a bucket; finite
    ones count up to 22180 either way, far beyond where a softmax tells them apart).  mask (B,n_k) or (n_k,),
    nonzero = real key.  q_start: position of query 0, default n_k - n_q (queries
    end where the keys end).  scale: default d ** -0.5.  Returns O like Q.
    """
    if not Q.is_cuda:
        out = flash_window_attn(_gpu(Q), _gpu(K), _gpu(V), window, sinks, causal, _gpu(pos_weight), buckets,
                                _gpu(mask), q_start, scale)
        return out.cpu()
    unbatched = Q.dim() == 3
    if unbatched:
        Q, K, V = Q.unsqueeze(0), K.unsqueeze(0), V.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
    if Q.dim() != 4 or K.dim() != 4:
        raise ValueError("Q must be (B, H, n_q, d) or (H, n_q, d), K and V alike")
    window, scale, lut, distance = _options(Q.shape[-1], window, sinks, scale, pos_weight, buckets, Q.device)
    q_start = K.shape[2] - Q.shape[2] if q_start is None else int(q_start)
    out = nat.ext().window_attn(Q, K, V, mask, pos_weight, lut, distance, window, min(int(sinks), 1 << 30),
                                bool(causal), q_start, scale)
    return out.squeeze(0) if unbatched else out


def window_attn_decode(q, k_cache, v_cache, lengths, window: int | None = None, sinks: int = 0,
                       pos_weight=None, buckets: RelativeBuckets | None = None, scale: float | None = None):
    """The newest token of each sequence: q (B,H,d) at position lengths[b] - 1, whose
    key and value are already in the cache.

    k_cache, v_cache (B,H_kv,n_max,d), any strides with unit stride along d;
    lengths (B,) int32 or int64 on the device, clamped to [0, n_max]; hidden rows
    (from lengths[b] on, or before the window) are never used, whatever they hold;
    a length of 0 gives zeros.  Returns (B,H,d).
    Forward only.
    """
    if not q.is_cuda:
        return window_attn_decode(_gpu(q), _gpu(k_cache), _gpu(v_cache), _gpu(lengths), window, sinks,
                                  _gpu(pos_weight), buckets, scale).cpu()
    if (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad
            or (pos_weight is not None and pos_weight.requires_grad)) and torch.is_grad_enabled():
        raise NotImplementedError("window_attn_decode is forward only: call it under torch.no_grad(), or "
                                  "flash_window_attn for gradients")
    window, scale, lut, distance = _options(q.shape[-1], window, sinks, scale, pos_weight, buckets, q.device)
    return nat.ext().window_attn_decode(q, k_cache, v_cache, lengths, pos_weight, lut, distance, window,
                                        min(int(sinks), 1 << 30), scale)
