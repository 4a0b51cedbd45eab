"""Position encodings on the GPU: the 68-bin position / bond code, and a learned
relative position bias by buckets.

``relative_position_bias`` (not in the reference, whose kernels look their 68
bins up themselves) gives the dense bias ``pos_weight[h, bucket(i + q_start - j)]``
and its gradient, e.g. to add to the cost of ``sinkhorn_solve``;
``flash_window_attn`` takes the same weights and buckets and never builds the
matrix.  ``RelativeBuckets`` holds the bucket of every distance.

``compute_bins``: drop-in for ``deepfold.model.position_encoding.compute_bins`` of the reference
(src/deepfold/model/position_encoding.py:7-52): same arguments, same (N, N) or
(B, N, N) int32 result,

    same chain, no bond:  clamp(global_idx_i - global_idx_j, -32, 32) + 32
    other chain, no bond: 65;  same chain, bond: 66;  other chain, bond: 67,

computed by the library (``dfs_compute_bins``).  The Sinkhorn operators can
skip the table altogether: pass ``pos_bins=(chain_id, global_idx,
bond_matrix)`` to ``flash_sinkhorn_attn`` / ``flash_sinkhorn`` and the kernels
evaluate each pair's bin where they use it.  CPU tensors are computed on the
current CUDA device and the result returned on the CPU (there is no CPU path).
"""

from __future__ import annotations

from array import array

import torch

from deepfold import _native as nat

__all__ = ["compute_bins", "RelativeBuckets", "relative_position_bias"]


def compute_bins(chain_id: torch.Tensor, global_idx: torch.Tensor, bond_matrix: torch.Tensor) -> torch.Tensor:
    """chain_id, global_idx (N,) or (B, N) int; bond_matrix (N, N) or (B, N, N)
    bool -> bins (N, N) or (B, N, N) int32 in [0, 67]."""
    unbatched = chain_id.dim() == 1
    if unbatched:
        chain_id, global_idx, bond_matrix = chain_id.unsqueeze(0), global_idx.unsqueeze(0), bond_matrix.unsqueeze(0)
    on_cpu = not chain_id.is_cuda
    if on_cpu:
        if not torch.cuda.is_available():
            raise RuntimeError("deepfold B200 ops run on a CUDA device; none is available (no CPU path)")
        dev = torch.device("cuda", torch.cuda.current_device())
        chain_id, global_idx, bond_matrix = chain_id.to(dev), global_idx.to(dev), bond_matrix.to(dev)
    bins = nat.ext().compute_bins(chain_id, global_idx, bond_matrix)
    if on_cpu:
        bins = bins.cpu()
    return bins.squeeze(0) if unbatched else bins


class RelativeBuckets:
    """The bucket of every relative distance delta = (query position) - (key position).

    ``table`` lists the buckets of delta = -D .. D (2 D + 1 whole numbers, D up to
    1024); its ends stand for all distances beyond.  A module keeps one of these
    beside its ``pos_weight`` (H, num_buckets); the device copy of the table is
    made once per device.
    """

    def __init__(self, table, num_buckets: int | None = None, device=None):
        table = list(map(int, table))
        if len(table) % 2 != 1 or len(table) > 2 * nat.DFS_MAX_BUCKET_DISTANCE + 1:
            raise ValueError("table must list the buckets of -D .. D: an odd number of them, D up to "
                             f"{nat.DFS_MAX_BUCKET_DISTANCE}")
        self.num_buckets = max(table) + 1 if num_buckets is None else int(num_buckets)
        if min(table) < 0 or max(table) >= self.num_buckets:
            raise ValueError(f"table entries must be in [0, {self.num_buckets})")
        self.max_distance = len(table) // 2
        self.table = tuple(table)
        self._on: dict[torch.device, torch.Tensor] = {}
        if device is not None:
            self.on(torch.device(device))

    @classmethod
    def clip(cls, max_distance: int = 32, device=None) -> "RelativeBuckets":
        """clamp(delta, -D, D) + D: ``compute_bins``' rule within a chain (65 buckets at D = 32)."""
        return cls(range(2 * max_distance + 1), device=device)

    @classmethod
    def log(cls, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True,
            device=None) -> "RelativeBuckets":
        """One bucket a distance up to half of a side's buckets, then
        logarithmically wider ones up to ``max_distance``, the last for all
        beyond.  ``bidirectional``: keys ahead (delta < 0) have the upper half of
        the buckets; else they share bucket 0.  The steps are found in whole
        numbers, so no rounding of a logarithm moves one."""
        side = num_buckets // 2 if bidirectional else num_buckets
        near = side // 2
        if near < 1 or max_distance <= near:
            raise ValueError("log buckets need num_buckets >= 4 (2 one-sided) and max_distance beyond the exact ones")
        wide = side - near

        def bucket(n: int) -> int:  # the largest step with (n / near)^wide >= (max_distance / near)^step
            if n < near:
                return n
            step = 0
            while step + 1 < wide and n ** wide * near ** (step + 1) >= max_distance ** (step + 1) * near ** wide:
                step += 1
            return near + step

        ahead = [num_buckets - side + bucket(n) if bidirectional else 0 for n in range(max_distance, 0, -1)]
        return cls(ahead + [bucket(n) for n in range(max_distance + 1)], num_buckets, device)

    def on(self, device: torch.device) -> torch.Tensor:
        """The table as int32 on ``device``."""
        t = self._on.get(device)
        if t is None:
            # an inference tensor, kept from a first call in inference mode, could not be saved for a later backward
            with torch.inference_mode(False):
                t = torch.frombuffer(array("i", self.table), dtype=torch.int32).to(device)  # quicker than from a list
            self._on[t.device] = self._on[device] = t
        return t


def check_buckets(pos_weight, buckets):
    """pos_weight (H, num_buckets) and buckets belong together."""
    if not isinstance(buckets, RelativeBuckets):
        raise TypeError("buckets must be a RelativeBuckets")
    if pos_weight.dim() != 2 or pos_weight.shape[1] != buckets.num_buckets:
        raise ValueError(f"pos_weight must be (H, {buckets.num_buckets}), the number of buckets; got "
                         f"{tuple(pos_weight.shape)}")


def relative_position_bias(pos_weight: torch.Tensor, buckets: RelativeBuckets, n_q: int, n_k: int,
                           q_start: int | None = None) -> torch.Tensor:
    """bias[h, i, j] = pos_weight[h, buckets(i + q_start - j)], (H, n_q, n_k) of pos_weight's type.

    q_start: position of the first query among the keys' positions; default
    ``n_k - n_q`` (queries and keys end together).  Differentiable in
    ``pos_weight``: the gradient sums over each bucket in fp32 and in a fixed
    order.
    """
    check_buckets(pos_weight, buckets)
    if n_q < 0 or n_k < 0:
        raise ValueError("n_q and n_k must not be negative")
    q_start = n_k - n_q if q_start is None else int(q_start)
    if not pos_weight.is_cuda:
        if not torch.cuda.is_available():
            raise RuntimeError("deepfold B200 ops run on a CUDA device; none is available (no CPU path)")
        dev = torch.device("cuda", torch.cuda.current_device())
        return relative_position_bias(pos_weight.to(dev), buckets, n_q, n_k, q_start).cpu()
    return nat.ext().relative_position_bias(pos_weight, buckets.on(pos_weight.device), buckets.max_distance,
                                            int(n_q), int(n_k), q_start)
