"""A linear layer without bias, out = x . W^T, with the kernel chosen by precision.

float32 engine: true 32-bit FMA (`csrc/gemm_f32.cu`) on float32 activations; the weight stays
as stored (bfloat16 is widened exactly inside the kernel).
A weight in 8 bits with a scale per block of 128 x 128 (`Fp8Weight`): in the bfloat16 engine the input is quantised per token and block of
128 columns, and the products run on the tensor cores in 8 bits (`csrc/gemm_fp8.cu`); the float32 engine takes what the weight stands for
into true 32-bit products.
bfloat16 engine: bfloat16 activations and weights with float32 accumulation on the tcgen05
tensor cores (`csrc/gemm_tc.cu`); a weight stored in float32, or a K that TMA cannot
address (not a multiple of 8), falls back to the SIMT kernel, which takes any size.

The tensor-core kernel cuts the K of a small weight into ranges (a function of the weight's shape
alone) whose sums are added in float32 in ascending order. With few tokens it leaves one partial
sum per range, so that the ranges run on different SMs; `forward_partials` and `forward_add` hand
those to the consumer (the rotation kernel, the next norm), which adds them. With many tokens the
kernel adds them itself, in the same order: a token's result has the same bits either way.
"""
from __future__ import annotations

import ctypes

import torch

from . import ops


FP8_SCALES = "_scale_inv"        # what the name of an 8-bit weight's scales in a checkpoint ends with


def fp8_scales_shape(rows: int, columns: int) -> tuple:
    return -(-rows // ops.FP8_BLOCK), -(-columns // ops.FP8_BLOCK)


def stack_rows(weights, compute_dtype: torch.dtype):
    """The matrices one below the other: tensors, or 8-bit weights (for the float32 engine what they stand for); of several kinds, all as float32."""
    weights = list(weights)
    if compute_dtype == torch.bfloat16 and all(isinstance(w, Fp8Weight) for w in weights):
        return Fp8Weight.stack(weights)
    weights = [w.to(torch.float32) if isinstance(w, Fp8Weight) else w for w in weights]
    if len({w.dtype for w in weights}) > 1:
        weights = [w.to(torch.float32) for w in weights]
    return torch.cat(weights, dim=0)


class Fp8Weight:
    """A [rows, columns] weight in e4m3 with one float32 scale per block of 128 rows and 128 columns: what it stands for is q * scale.
    q float8_e4m3fn; scales [ceil(rows / 128), ceil(columns / 128)]. Rows are kept 16-byte aligned (`stride` bytes apart)."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, halves: int = 1, in_blocks: bool = True):
        if q.dim() != 2 or q.dtype != torch.float8_e4m3fn:
            raise TypeError("an 8-bit weight is a [out, in] matrix of float8_e4m3fn")
        M, K = q.shape
        rows = halves * -(-(M // halves) // ops.FP8_BLOCK)
        if scales.dim() != 2 or tuple(scales.shape) != (rows, -(-K // ops.FP8_BLOCK)) or scales.dtype != torch.float32:
            raise ValueError(f"the scales of a {M} x {K} weight are float32 [{rows}, {-(-K // ops.FP8_BLOCK)}], not {scales.dtype} {list(scales.shape)}")
        if scales.device != q.device:
            raise ValueError(f"an 8-bit weight on {q.device} has its scales there too, not on {scales.device}")
        self.shape = (M, K)
        self.stride = -(-K // 16) * 16
        if q.stride(0) == self.stride and (K == 1 or q.stride(1) == 1) and q.data_ptr() % 16 == 0 and self.stride == K:
            self.q = q
        else:
            self.q = torch.zeros(M, self.stride, dtype=torch.uint8, device=q.device)
            self.q[:, :K] = q.view(torch.uint8)
            self.q = self.q.view(torch.float8_e4m3fn)
        self.scales = scales.contiguous()
        self.halves, self.in_blocks = halves, in_blocks

    @property
    def dtype(self):
        return torch.float8_e4m3fn

    @property
    def device(self):
        return self.q.device

    def nbytes(self) -> int:
        return self.shape[0] * self.shape[1] + 4 * self.scales.numel()

    @staticmethod
    def stack(weights) -> "Fp8Weight":
        """The matrices one below the other. Blocks of scales begin anew with every matrix: unless all but the last have a multiple of 128 rows, the
        result can only be the [gate rows; up rows] of a gated product, two matrices of one shape."""
        weights = list(weights)
        if len(weights) == 1:
            return weights[0]
        if any(w.halves != 1 or not w.in_blocks for w in weights) or len({w.shape[1] for w in weights}) > 1:
            raise ValueError("stacked 8-bit weights are plain matrices with the same number of columns")
        halves = 2 if len(weights) == 2 and weights[0].shape == weights[1].shape else 1
        in_blocks = all(w.shape[0] % ops.FP8_BLOCK == 0 for w in weights[:-1])
        if halves == 1 and not in_blocks:
            raise ValueError(f"8-bit matrices of {[w.shape[0] for w in weights]} rows cannot be stacked: their scales cover 128 rows each")
        K = weights[0].shape[1]
        q = torch.cat([w.q.view(torch.uint8) for w in weights]).view(torch.float8_e4m3fn)
        return Fp8Weight(q[:, :K], torch.cat([w.scales for w in weights]), halves, in_blocks)

    @staticmethod
    def quantize(weight: torch.Tensor) -> "Fp8Weight":
        """A matrix rounded to this form: scale = max |w| of the block / 448 (1 for a block of zeros), q = e4m3(w / scale)."""
        M, K = weight.shape
        B = ops.FP8_BLOCK
        padded = torch.zeros(-(-M // B) * B, -(-K // B) * B, dtype=torch.float32, device=weight.device)
        padded[:M, :K] = weight
        blocks = padded.view(padded.shape[0] // B, B, padded.shape[1] // B, B)
        scales = blocks.abs().amax(dim=(1, 3)) / 448.0
        scales = torch.where(scales > 0, scales, torch.ones_like(scales))
        q = (blocks / scales[:, None, :, None]).clamp(-448.0, 448.0).reshape(padded.shape)[:M, :K].to(torch.float8_e4m3fn)
        return Fp8Weight(q, scales)

    def to(self, dtype: torch.dtype) -> torch.Tensor:
        """The matrix that it stands for, in float32 (each element rounded once) or a narrower type."""
        M, K = self.shape
        B = ops.FP8_BLOCK
        half = M // self.halves
        rows = torch.arange(M, device=self.device)
        block = (rows // half) * -(-half // B) + (rows % half) // B
        scales = self.scales[block].repeat_interleave(B, 1)[:, :K]
        return (self.q[:, :K].to(torch.float32) * scales).to(dtype)


class Fp8Experts:
    """Gated experts with 8-bit weights, laid out for `ops.experts_fp8`. gate_up: gate and up matrix of every expert in turn ([inner, width] each);
    down: every expert's [width, inner]."""

    def __init__(self, gate_up, down):
        gate_up, down = list(gate_up), list(down)
        shapes = {w.shape for w in gate_up}, {w.shape for w in down}
        if len(gate_up) != 2 * len(down) or not down or len(shapes[0]) != 1 or len(shapes[1]) != 1 or down[0].shape != gate_up[0].shape[::-1]:
            raise ValueError("experts have a gate and an up matrix [inner, width] and a down matrix [width, inner] each")
        if not all(w.in_blocks for w in gate_up + down):
            raise ValueError("an expert's matrices are plain ones: blocks of scales that begin anew in the middle of one are not laid out so")
        if len({w.device for w in gate_up + down}) != 1:
            raise ValueError("the experts' matrices are all on one device")
        self.experts = len(down)
        self.inner, self.width = gate_up[0].shape
        self.gate_up = torch.cat([w.q.view(torch.uint8) for w in gate_up]).view(torch.float8_e4m3fn)
        self.gate_up_scales = torch.cat([w.scales for w in gate_up])
        self.down = torch.cat([w.q.view(torch.uint8) for w in down]).view(torch.float8_e4m3fn)
        self.down_scales = torch.cat([w.scales for w in down])
        self._layout = ops._Fp8ExpertsLayout(self.gate_up.data_ptr(), self.gate_up.stride(0), self.gate_up_scales.data_ptr(), self.down.data_ptr(),
                                             self.down.stride(0), self.down_scales.data_ptr(), self.experts, self.width, self.inner)
        self.address = ctypes.addressof(self._layout)
        self.at = self.down.get_device()          # -1: not on a CUDA device

    def weight_bytes(self) -> int:
        """Of one expert."""
        return (3 * self.inner * self.width) + 4 * (self.gate_up_scales.numel() + self.down_scales.numel()) // self.experts

    def scratch(self, n: int, top: int) -> torch.Tensor:
        return torch.empty(ops.experts_fp8_scratch(n, top, self.experts, self.width, self.inner), dtype=torch.uint8, device=self.down.device)

    def forward(self, x: torch.Tensor, choice: torch.Tensor, weights: torch.Tensor, out: torch.Tensor, scratch: torch.Tensor) -> None:
        ops.experts_fp8(x, choice, weights, self, out, scratch)


class Linear:
    def __init__(self, weight, compute_dtype: torch.dtype):
        if isinstance(weight, Fp8Weight) and compute_dtype != torch.bfloat16:
            weight = weight.to(torch.float32)          # the 32-bit engine: what the 8-bit weight stands for, in true 32-bit products
        self.fp8 = weight if isinstance(weight, Fp8Weight) else None
        if self.fp8 is not None:
            self.weight = self._call = self._call_workspace = None
            self.out_features, self.in_features = weight.shape
            self.compute_dtype, self.tensor_core, self.splits = compute_dtype, False, 1
            return
        if weight.dim() != 2:
            raise ValueError("Linear takes a [out, in] matrix")
        self.weight = weight.contiguous()
        self.out_features, self.in_features = weight.shape
        self.compute_dtype = compute_dtype
        self.tensor_core = (compute_dtype == torch.bfloat16 and self.weight.dtype == torch.bfloat16
                            and self.in_features % 8 == 0)
        self.splits = ops.gemm_tc_splits(self.out_features, self.in_features) if self.tensor_core else 1

    def weight_bytes(self) -> int:
        return self.fp8.nbytes() if self.fp8 is not None else self.weight.numel() * self.weight.element_size()

    def _buffers(self, workspace):
        """The workspace's buffers for the quantised rows of this layer's input: (values, scales)."""
        if workspace is None:
            raise ValueError("a linear layer with an 8-bit weight takes the workspace that its quantised input is kept in")
        T, K = workspace.max_tokens, self.in_features
        q = workspace.raw("linear.fp8", (T, -(-K // 16) * 16), torch.float8_e4m3fn)
        return q, workspace.raw("linear.fp8_scales", (-(-K // ops.FP8_BLOCK), T), torch.float32)

    def _fp8(self, x: torch.Tensor, out: torch.Tensor, epilogue: int, workspace, constants=(0.0, 0.0)) -> None:
        if self._call is None or self._call_workspace is not workspace:
            self._call, self._call_workspace = ops.Fp8Linear(self.fp8, *self._buffers(workspace)), workspace
        self._call(x, out, epilogue, constants)

    def _tc(self, x: torch.Tensor) -> bool:
        return self.tensor_core and x.dtype == torch.bfloat16 and x.stride(0) % 8 == 0

    def partial_elems(self, max_tokens: int) -> int:
        """Elements of the largest partial buffer `forward_partials` may need for up to max_tokens tokens."""
        rows = max_tokens
        if self.tensor_core:
            rows = max(rows, min(max_tokens, ops.gemm_tc_partial_tokens()) * self.splits)
        return rows * self.out_features

    def forward(self, x: torch.Tensor, out: torch.Tensor, workspace=None) -> None:
        """out[n, out_features] float32 = x . W^T, K in one range whatever the weight's shape (an 8-bit weight: out may be bfloat16, K is cut by the
        weight's shape, `workspace` holds the quantised input)."""
        if self.fp8 is not None:
            self._fp8(x, out, ops.STORE, workspace)
        elif self._tc(x):
            ops.gemm_tc(x, self.weight, out, ops.STORE)
        else:
            ops.gemm_f32(x, self.weight, out, accumulate=False)

    def forward_partials(self, x: torch.Tensor, flat: torch.Tensor, workspace=None) -> torch.Tensor:
        """x . W^T as [S, n, out_features] float32 partial sums (S >= 1) carved from the flat buffer `flat`."""
        n, M = x.shape[0], self.out_features
        if self.fp8 is not None:
            out = flat[:n * M].view(1, n, M)
            self._fp8(x, out[0], ops.STORE, workspace)
            return out
        if not self._tc(x):
            out = flat[:n * M].view(1, n, M)
            ops.gemm_f32(x, self.weight, out[0], accumulate=False)
            return out
        S = self.splits if n <= ops.gemm_tc_partial_tokens() else 1     # buffers left; the ranges stay the same
        out = flat[:S * n * M].view(S, n, M)
        ops.gemm_tc(x, self.weight, out if S > 1 else out[0], ops.STORE, splits=self.splits)
        return out

    def forward_add(self, x: torch.Tensor, stream, flat: torch.Tensor = None, workspace=None) -> None:
        """stream += x . W^T (the residual add). With `flat` given, K is cut into the weight's ranges and, for few
        tokens, their partial sums are left pending on the stream; without it K stays one range. A call site
        must choose one of the two for good: the order of the sums differs."""
        if self.fp8 is not None:
            stream.fold()
            self._fp8(x, stream.h, ops.ADD, workspace)
        elif self._tc(x):
            n, M, S = x.shape[0], self.out_features, self.splits if flat is not None else 1
            if S > 1:
                # few tokens: one partial sum per range; many: the ranges' sum. Either way the stream's next
                # consumer computes h + (range_0 + range_1 + ...).
                P = S if n <= ops.gemm_tc_partial_tokens() else 1
                parts = flat[:P * n * M].view(P, n, M)
                ops.gemm_tc(x, self.weight, parts if P > 1 else parts[0], ops.STORE, splits=S)
                stream.set_pending(parts)
                return
            stream.fold()
            ops.gemm_tc(x, self.weight, stream.h, ops.ADD)
        else:
            stream.fold()
            ops.gemm_f32(x, self.weight, stream.h, accumulate=True)

    # ------------------------------------------------------------------ the same, as operations of the native step program
    # (`x`, `out`, `flat`, `z` are the full buffers, of which a step uses its first n rows)
    def _f32_op(self, program, x, out, ldo: int, accumulate: bool, wanted_rows: bool) -> None:
        program.add("gemm_f32", "sb_op_linear_f32", [x, x.dtype, x.stride(0), self.weight, self.weight.dtype, self.weight.stride(0), out, ldo,
                                                      self.out_features, self.in_features, int(accumulate), int(wanted_rows)])

    def _tc_op(self, program, x, out, mode: int, splits: int = 1, wanted_rows: bool = False, constants=()) -> None:
        # the decode chain has phases for partial sums per K range and for SwiGLU, on the step's tokens
        phase = None
        if not wanted_rows and mode in (1, 3):      # (the chain's gated epilogue is silu's: modes 4 and 5 have no phase)
            phase = lambda chain: chain.linear(x, self.weight, out, mode == 3, splits if mode == 1 else 1)
        program.add("gemm_tc", "sb_op_linear_tc", [x, x.stride(0), self.weight, self.weight.stride(0), out, self.out_features,
                                                    self.in_features, mode, splits, int(wanted_rows)], constants, chain=phase)

    def _fp8_op(self, program, x, out, ldo: int, epilogue: int, wanted_rows: bool = False, act: int = 0, constants=()) -> None:
        q, scales = self._buffers(program.workspace)
        w = self.fp8
        ops.check_fp8_epilogue(w, epilogue == 2)
        program.add("gemm_fp8", "sb_op_linear_fp8", [q, q.stride(0), scales, scales.stride(0), w.q, w.stride, w.scales, *w.shape, w.shape[0] // 2,
                                                     x, x.dtype, x.stride(0), out, out.dtype, ldo, epilogue, act, int(wanted_rows)], constants)

    def emit(self, program, x: torch.Tensor, out: torch.Tensor, wanted_rows: bool = False) -> None:
        """`forward`; with `wanted_rows` the rows are the step's wanted rows (the head), not its tokens."""
        if self.fp8 is not None:
            self._fp8_op(program, x, out, out.stride(0), 0, wanted_rows)
        elif self._tc(x):
            self._tc_op(program, x, out, 0, wanted_rows=wanted_rows)
        else:
            self._f32_op(program, x, out, out.stride(0), False, wanted_rows)

    def emit_partials(self, program, x: torch.Tensor, flat: torch.Tensor) -> int:
        """`forward_partials`; returns the number of K ranges S that the reader of `flat` has to expect
        ([S, n, out_features] up to `program.few_tokens` tokens, [1, n, out_features] beyond)."""
        if self.fp8 is not None:
            self._fp8_op(program, x, flat, self.out_features, 0)
            return 1
        if not self._tc(x):
            self._f32_op(program, x, flat, self.out_features, False, False)
            return 1
        self._tc_op(program, x, flat, 1, self.splits)
        return self.splits

    def emit_add(self, program, x: torch.Tensor, flat: torch.Tensor = None) -> None:
        """`forward_add` onto the program's residual stream."""
        if self._tc(x) and flat is not None and self.splits > 1:
            program.need_folded("a projection that leaves partial sums")
            self._tc_op(program, x, flat, 1, self.splits)
            program.pending = (flat, self.splits, self.out_features)
            return
        program.need_folded("a projection")
        fresh = program.take_fresh()        # a branch that holds nothing yet: the result is stored, not added
        if fresh is not None:
            return self.emit(program, x, fresh)
        if self.fp8 is not None:
            self._fp8_op(program, x, program.h, program.h.stride(0), 1)
        elif self._tc(x):
            self._tc_op(program, x, program.h, 2)
        else:
            self._f32_op(program, x, program.h, program.h.stride(0), True, False)

    def emit_swiglu(self, program, x: torch.Tensor, z: torch.Tensor, scratch_fn, activation: str = "silu", constants=()) -> None:
        """`forward_swiglu`."""
        act = ops.GATE_ACTIVATIONS[activation]
        if self.fp8 is not None:
            self._fp8_op(program, x, z, z.stride(0), 2, act=act, constants=constants)
        elif self._tc(x) and z.dtype == torch.bfloat16:
            self._tc_op(program, x, z, 3 + act, constants=constants)
        else:
            gate_up = scratch_fn()
            self._f32_op(program, x, gate_up, gate_up.stride(0), False, False)
            program.add("elementwise", "sb_op_swiglu", [gate_up, z, z.dtype, self.out_features // 2, act], constants)

    def forward_swiglu(self, x: torch.Tensor, z: torch.Tensor, scratch_fn, activation: str = "silu", constants=(), workspace=None) -> None:
        """W = [gate rows; up rows]: z[n, I] = act(x . gate^T) * (x . up^T), act = silu or the tanh form of gelu, or the clamped gate with
        its constants (`ops.swiglu`).
        `scratch_fn()` gives a float32 [n, 2 I] buffer for the unfused path."""
        I = self.out_features // 2
        if self.fp8 is not None:
            self._fp8(x, z, ops.SWIGLU + ops.GATE_ACTIVATIONS[activation], workspace, constants or (0.0, 0.0))
        elif self._tc(x) and z.dtype == torch.bfloat16:
            ops.gemm_tc(x, self.weight, z, ops.SWIGLU + ops.GATE_ACTIVATIONS[activation], half_rows=I, constants=constants or (0.0, 0.0))
        else:
            gate_up = scratch_fn()
            ops.gemm_f32(x, self.weight, gate_up, accumulate=False)
            ops.swiglu(gate_up, z, activation, constants or (0.0, 0.0))
