"""A mixture of experts over INT4 weights: routing, the experts' products and
their combination.

    r = route(logits, top_k=8)                       # [T, E] -> experts, order
    h = gate_up(x, r, activation="silu", gated=True)  # [T * 8, F], expert order
    y = down(h, r, gather=False)                     # [T * 8, N], expert order
    out = combine(y, r, residual=x)                  # [T, N]

(``ExpertMLP`` is those four calls.) Nothing is read back to the host: the
number of rows an expert gets stays on the device, and every buffer has
T * top_k rows whatever the routing is. Rows behind the last expert's (tokens
routed to fewer than top_k experts) are left as they were.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import (ACTIVATIONS, GROUP_SCORES, SCORINGS, launch_quantize_repack,
               launch_repack_scales_128, launch_repack_umma)
from .launching import binding, cuda_device, on
from .linear import interleave_gate_up


class Routing(NamedTuple):
    """A batch's routing (from `route`: five tensors in one allocation). A pair is
    token * top_k + place."""
    ids: torch.Tensor      # int32 [T, top_k]: experts, best first (-1: none)
    weights: torch.Tensor  # float32 [T, top_k]
    offsets: torch.Tensor  # int32 [E + 1]: expert e has sorted rows offsets[e] .. offsets[e + 1]
    rows: torch.Tensor     # int32 [T * top_k]: the pair of each sorted row (-1 past the last)
    slots: torch.Tensor    # int32 [T, top_k]: the sorted row of each pair (-1: none)


def route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax",
          bias: torch.Tensor | None = None, n_group: int = 1, topk_group: int = 1,
          group_score: str = "max", renormalize: bool = True, scale: float = 1.0,
          stream=None) -> Routing:
    """Each token's ``top_k`` experts from its logits [T, E] (float32 or
    float16, rows of any stride), as C ABI i4g_route describes: softmax or
    sigmoid scores, ``bias`` (float32 [E]) added for the choice only, the best
    ``topk_group`` of ``n_group`` groups, ties to the lowest index, weights
    renormalised to sum 1 and scaled."""
    kind, of_group = SCORINGS.get(scoring), GROUP_SCORES.get(group_score)
    if kind is None or of_group is None:
        raise ValueError(f"unknown scoring {scoring!r} or group_score {group_score!r}")
    dev = cuda_device(logits, "logits")
    with on(dev, stream, logits, bias):
        return Routing(*binding().route(logits, top_k, kind, bias, n_group, topk_group, of_group,
                                        renormalize, scale))


def combine(y: torch.Tensor, routing: Routing, *, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """out[t] = residual[t] + sum over places s of weights[t, s] * y[slots[t, s]]
    (C ABI i4g_experts_combine): y fp16 in expert order, out fp16 [T, N]."""
    dev = cuda_device(y, "y")
    with on(dev, stream, y, routing.weights, routing.slots, residual, out):
        return binding().combine(y, routing.slots, routing.weights, residual, out)


class QuantizedExperts:
    """E experts' INT4 weights of one [K, N], one after another in the GEMM's layouts."""

    def __init__(self, tiles: torch.Tensor, scales: torch.Tensor, E: int, K: int, N: int,
                 group: int):
        if tiles.dtype != torch.uint8 or scales.dtype != torch.float16:
            raise TypeError("tiles must be uint8 and scales float16")
        if tiles.numel() != E * (K * N // 2) or scales.numel() != E * (K // group) * N:
            raise ValueError("buffer sizes do not match E, K, N, group")
        if not tiles.is_contiguous() or not scales.is_contiguous():
            raise ValueError("tiles and scales must be contiguous")
        self.tiles, self.scales = tiles.view(E, -1), scales.view(E, -1)
        self.E, self.K, self.N, self.group = E, K, N, group

    @classmethod
    def _empty(cls, E, K, N, group, device):
        tiles = torch.empty(E, K * N // 2, dtype=torch.uint8, device=device)
        scales = torch.empty(E, (K // group) * N, dtype=torch.float16, device=device)
        return cls(tiles, scales, E, K, N, group)

    @classmethod
    def from_weight(cls, w: torch.Tensor, group: int, stream=None) -> "QuantizedExperts":
        """Quantise fp16 [E, K, N] weights, each as QuantizedLinear.from_weight does."""
        dev = cuda_device(w, "weight")
        if w.dtype != torch.float16 or w.dim() != 3:
            raise TypeError("weight must be a 3-D float16 CUDA tensor [E, K, N]")
        E, K, N = w.shape
        with on(dev, stream, w):
            self = cls._empty(E, K, N, group, dev)
            for e in range(E):
                launch_quantize_repack(w[e].contiguous(), self.tiles[e], self.scales[e], K, N,
                                       group)
        return self

    @classmethod
    def from_gate_up(cls, gate: torch.Tensor, up: torch.Tensor, group: int,
                     stream=None) -> "QuantizedExperts":
        """One weight per expert of the fp16 [E, K, F] gate and up projections, for
        calls with gated=True."""
        dev = cuda_device(gate, "gate")
        with on(dev, stream, gate, up):  # the joined weights belong to the stream that reads them
            return cls.from_weight(interleave_gate_up(gate, up), group)

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor, K: int, N: int, group: int,
                    stream=None) -> "QuantizedExperts":
        """Repack quantiser-layout codes [E][K * N / 2] and scales [E][K / group][N]."""
        E, dev = packed.shape[0], cuda_device(packed, "packed")
        if packed.dtype != torch.uint8 or scales.dtype != torch.float16 or scales.device != dev:
            raise TypeError("packed must be uint8 and scales float16, on one device")
        if packed.numel() != E * (K * N // 2) or scales.numel() != E * (K // group) * N:
            raise ValueError("buffer sizes do not match E, K, N, group")
        with on(dev, stream, packed, scales):
            self = cls._empty(E, K, N, group, dev)
            packed, scales = packed.contiguous().view(E, -1), scales.contiguous().view(E, -1)
            for e in range(E):
                launch_repack_umma(packed[e], self.tiles[e], K, N)
                launch_repack_scales_128(scales[e], self.scales[e], K, N, group)
        return self

    def __call__(self, a: torch.Tensor, routing: Routing, *, gather: bool = True,
                 bias: torch.Tensor | None = None, activation: str = "none", gated: bool = False,
                 out: torch.Tensor | None = None, fp32_out: bool = False,
                 stream=None) -> torch.Tensor:
        """The routed rows' products in expert order, [T * top_k, N] (gated: N / 2).
        gather: ``a`` is the tokens' rows [T, K]; otherwise rows already in
        expert order [T * top_k, K]. bias: fp16 [E, N]. Rows of the result past
        routing.offsets[E] are left as they were."""
        kind = ACTIVATIONS.get(activation)
        if kind is None:
            raise ValueError(f"unknown activation {activation!r}")
        dev = cuda_device(self.tiles, "the weights")
        with on(dev, stream, self.tiles, self.scales, a, routing.offsets, routing.rows, bias, out):
            return binding().experts_gemm(a, self.tiles, self.scales, self.E, self.K, self.N,
                                          self.group, routing.offsets, routing.rows,
                                          routing.slots, gather, bias, kind, gated, out, fp32_out)


class ExpertMLP:
    """The gated MLP of a mixture of experts: gate and up projection
    (``gate_up``: K -> 2 F, columns of ``from_gate_up``), activation, ``down``:
    F -> K, weighted sum."""

    def __init__(self, gate_up: QuantizedExperts, down: QuantizedExperts,
                 activation: str = "silu"):
        if gate_up.E != down.E or gate_up.N != 2 * down.K:
            raise ValueError("gate_up [E, K, 2 F] and down [E, F, N] do not belong together")
        self.gate_up, self.down, self.activation = gate_up, down, activation

    def __call__(self, x: torch.Tensor, routing: Routing, *,
                 residual: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        h = self.gate_up(x, routing, activation=self.activation, gated=True, stream=stream)
        y = self.down(h, routing, gather=False, stream=stream)
        return combine(y, routing, residual=residual, stream=stream)

