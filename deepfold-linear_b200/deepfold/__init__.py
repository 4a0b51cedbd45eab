"""B200-native drop-in for the flash-Sinkhorn path of DeepFold-Linear.

Mirrors the reference package layout for that path, with local attention beside it:

* ``deepfold.model.kernels.flash_sinkhorn_attn.flash_sinkhorn_attn``
* ``deepfold.model.kernels.sinkhorn_kernel.flash_sinkhorn``
* ``deepfold.model.sinkhorn.sinkhorn_solve``
* ``deepfold.model.kernels.flash_window_attn.flash_window_attn`` /
  ``window_attn_decode`` and ``deepfold.model.position_encoding.
  relative_position_bias`` -- local softmax attention and its position bias
  (new here: not drop-ins for the reference's softmax attention)
* ``deepfold.utils.cg.conjugate_gradient`` / ``steihaug_cg``
* ``deepfold.sharding`` -- multi-GPU (batch, head) and row sharding

All Sinkhorn compute runs in ``libdfsink.so`` (hand-written sm_100a CUDA behind
the C ABI of ``include/dfsink.h``).
"""

__version__ = "0.1.0"
