"""A quantised weight held in the sm_100a layouts, and its GEMM.

Owns the two device buffers the fused GEMM reads: the tile-layout INT4 codes
(``launch_repack_umma``) and the 128-column scale layout
(``launch_repack_scales_128``). Column-parallel shards are zero-copy views:
a rank's columns are one contiguous byte range of each buffer.
"""
from __future__ import annotations

import torch

from . import (ACTIVATIONS, launch_final_fp32_ws, launch_final_ws, launch_quantize_repack,
               launch_repack_scales_128, launch_repack_umma, shard_range, workspace_for)
from .launching import binding, cuda_device, mark, on


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """[..., F] gates and ups -> [..., 2 F] gated columns: groups of 16, eight
    gates and then the eight columns they gate (weights or biases)."""
    if gate.shape != up.shape or gate.shape[-1] % 8:
        raise ValueError("gate and up need one shape and a multiple of 8 columns")
    lead, F = gate.shape[:-1], gate.shape[-1]
    both = torch.stack((gate.reshape(*lead, F // 8, 8), up.reshape(*lead, F // 8, 8)), dim=-2)
    return both.reshape(*lead, 2 * F)


class QuantizedLinear:
    def __init__(self, tiles: torch.Tensor, scales: torch.Tensor, K: int, N: int, group: int):
        if tiles.dtype != torch.uint8 or scales.dtype != torch.float16:
            raise TypeError("tiles must be uint8 and scales float16")
        if tiles.numel() != K * N // 2 or scales.numel() != (K // group) * N:
            raise ValueError("buffer sizes do not match K, N, group")
        self.tiles, self.scales = tiles, scales
        self.K, self.N, self.group = K, N, group

    @classmethod
    def from_weight(cls, w: torch.Tensor, group: int, stream=None) -> "QuantizedLinear":
        """Quantise an fp16 [K, N] weight on the GPU (codes and scales
        bit-identical to the reference's quantize_cpu) straight into the GEMM
        layouts, in one pass."""
        if w.dtype != torch.float16 or w.dim() != 2 or not w.is_cuda:
            raise TypeError("weight must be a 2-D float16 CUDA tensor [K, N]")
        K, N = w.shape
        dev = w.device
        with on(dev, stream, w):
            tiles = torch.empty(K * N // 2, dtype=torch.uint8, device=dev)
            rscales = torch.empty((K // group) * N, dtype=torch.float16, device=dev)
            launch_quantize_repack(w.contiguous(), tiles, rscales, K, N, group)
        return cls(tiles, rscales, K, N, group)

    @classmethod
    def from_gate_up(cls, gate: torch.Tensor, up: torch.Tensor, group: int,
                     stream=None) -> "QuantizedLinear":
        """One weight of the fp16 [K, F] gate and up projections, for calls with
        gated=True (F % 64 == 0; a column's codes do not depend on its place)."""
        dev = cuda_device(gate, "gate")
        with on(dev, stream, gate, up):  # the joined weight belongs to the stream that reads it
            return cls.from_weight(interleave_gate_up(gate, up), group)

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor, K: int, N: int,
                    group: int, stream=None) -> "QuantizedLinear":
        """Repack reference-layout codes ([K][N] nibbles) and scales ([K/g][N])."""
        dev = cuda_device(packed, "packed")
        with on(dev, stream, packed, scales):
            tiles = torch.empty(K * N // 2, dtype=torch.uint8, device=dev)
            rscales = torch.empty((K // group) * N, dtype=torch.float16, device=dev)
            launch_repack_umma(packed, tiles, K, N)
            launch_repack_scales_128(scales, rscales, K, N, group)
        return cls(tiles, rscales, K, N, group)

    def shard(self, world: int, rank: int) -> "QuantizedLinear":
        """This rank's column slice of a world-way column-parallel split (a view)."""
        toff, soff, n0, n1 = shard_range(self.K, self.N, self.group, world, rank)
        n_local = n1 - n0
        tiles = self.tiles[toff: toff + self.K * n_local // 2]
        s0 = soff // 2
        scales = self.scales[s0: s0 + (self.K // self.group) * n_local]
        return QuantizedLinear(tiles, scales, self.K, n_local, self.group)

    def __call__(self, a: torch.Tensor, out: torch.Tensor | None = None, fp32_out: bool = False,
                 stream=None, *, bias: torch.Tensor | None = None, activation: str = "none",
                 gated: bool = False, residual: torch.Tensor | None = None) -> torch.Tensor:
        """A x dequant(B), or with any of the keyword arguments the fused epilogue
        (``launch_final_epilogue``): act(A x dequant(B) + bias) + residual, and with
        ``gated`` (columns as ``from_gate_up`` lays them out) act(gate) * up with N / 2
        columns. bias: fp16 [N]; residual: fp16, C's shape, rows of any stride (it may be
        ``out``)."""
        if bias is not None or residual is not None or gated or activation != "none":
            return self._epilogue(a, out, fp32_out, stream, bias, activation, gated, residual)
        if a.dtype != torch.float16 or a.dim() != 2 or a.shape[1] != self.K:
            raise ValueError(f"A must be float16 [M, {self.K}]")
        M = a.shape[0]
        dtype = torch.float32 if fp32_out else torch.float16
        if stream is not None:
            s = mark(self.tiles.device, stream, self.tiles, self.scales, a, out)
            if out is None or not a.is_contiguous():  # made on the stream, and its own
                with torch.cuda.stream(s):
                    a = a.contiguous()
                    out = torch.empty(M, self.N, dtype=dtype, device=a.device) if out is None else out
        else:
            a = a.contiguous()
            if out is None:
                out = torch.empty(M, self.N, dtype=dtype, device=a.device)
        ws = workspace_for(M, self.N, self.K, a.device, stream)
        fn = launch_final_fp32_ws if fp32_out else launch_final_ws
        fn(a, self.tiles, self.scales, out, M, self.N, self.K, self.group, ws, stream)
        return out

    def _epilogue(self, a, out, fp32_out, stream, bias, activation, gated, residual):
        kind = ACTIVATIONS.get(activation)
        if kind is None:
            raise ValueError(f"unknown activation {activation!r}")
        dev = cuda_device(self.tiles, "the weight")
        with on(dev, stream, self.tiles, self.scales, a, bias, residual, out):
            return binding().gemm_epilogue(a, self.tiles, self.scales, self.K, self.N, self.group,
                                           bias, kind, gated, residual, out, fp32_out)
