"""torch-ROCm front of the C ABI: shape/dtype checks, output allocation, launch.

Every function takes device tensors, checks them against what the kernel and
its grid assume (on the host, before anything is enqueued), allocates the
outputs with torch (Python owns all buffers), and enqueues the kernel on the
current stream. No function here computes anything on the CPU.
"""

from __future__ import annotations

import contextlib
import ctypes
import warnings
from typing import NamedTuple

import torch

from . import _lib

BF16 = torch.bfloat16


# A decode step's kernels run 2-5 us each and its launches come from here one by one, so the checks
# cost what they must and no more: raw stream handles and addresses (ctypes takes plain ints), one pass
# over a tensor's attributes, and the reasons only for a tensor that fails (the 896-wide decoder's
# prefill and functional step: 4112 -> 2707 us; one projection, allocation included: 13.1 -> 8.9 us).
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _stream(device: int | None = None) -> int:
    """The current device's stream (``device``: that device's number, where the caller has it)."""

    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device() if device is None else device)


def _ptr(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()


def _expect(tensor: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple[int, ...] | None = None) -> None:
    if (isinstance(tensor, torch.Tensor) and tensor.is_cuda and tensor.dtype is dtype and tensor.is_contiguous()
            and (shape is None or tensor.shape == shape)):
        return
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(tensor).__name__}")
    if tensor.device.type != "cuda":
        raise ValueError(f"{name} must be on the GPU, got {tensor.device}")
    if tensor.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {tensor.dtype}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(tensor.shape)}")


def _on_device(workspace: torch.Tensor | None) -> None:
    """A workspace in host memory is an illegal access for the kernel that stores its partial sums there."""

    if workspace is not None and not workspace.is_cuda:
        raise ValueError(f"the workspace must be on a GPU, got {workspace.device}")


def _ready(tensor: torch.Tensor) -> None:
    _lib.ensure_code_object(tensor.get_device())


#: codes per packed int32 word of each width
CODES_PER_WORD = {4: 8, 8: 4}


def take_launches() -> list[str]:
    """Kernel symbols this thread launched since the last call, while :func:`recording_launches`
    is active (``aoto_hip_take_launches``)."""

    lib = _lib.library()
    size = int(lib.aoto_hip_take_launches(None, 0))
    if size == 0:
        return []
    buf = ctypes.create_string_buffer(size + 1)
    lib.aoto_hip_take_launches(buf, size + 1)
    return buf.value.decode().split()


@contextlib.contextmanager
def recording_launches(*, only: bool = False):
    """Record the kernel symbols this thread launches (read them with :func:`take_launches`).

    ``only=True`` records what it would launch and launches nothing.
    """

    lib = _lib.library()
    previous = int(lib.aoto_hip_trace_launches(2 if only else 1))
    try:
        yield take_launches
    finally:
        if not previous:
            take_launches()
        lib.aoto_hip_trace_launches(previous)


def _quantize(weight: torch.Tensor, group_size: int, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    per_word = CODES_PER_WORD[bits]
    if weight.dim() != 2:
        raise ValueError(f"a quantized weight must be 2-D, got {tuple(weight.shape)}")
    if weight.dtype not in (BF16, torch.float32):
        raise TypeError(f"weight must be bf16 or f32, got {weight.dtype}")
    _expect(weight, "weight", weight.dtype)
    rows, inner = weight.shape
    if group_size <= 0 or group_size % per_word or inner % group_size:
        raise ValueError(f"group size {group_size} must be a positive multiple of {per_word} dividing {inner}")
    _ready(weight)
    packed = torch.empty((rows, inner // per_word), dtype=torch.int32, device=weight.device)
    scales = torch.empty((rows, inner // group_size), dtype=BF16, device=weight.device)
    entry = _lib.library().aoto_hip_w4_quantize if bits == 4 else _lib.library().aoto_hip_w8_quantize
    _lib.check(
        entry(
            _ptr(weight), int(weight.dtype == torch.float32), rows, inner, group_size,
            _ptr(packed), _ptr(scales), None, _stream(),
        )
    )
    return packed, scales


def w4_quantize(weight: torch.Tensor, group_size: int = 64) -> tuple[torch.Tensor, torch.Tensor]:
    """Pack a ``[out, in]`` bf16/f32 weight: ``(int32 [out, in/8], bf16 scales [out, in/group])``.

    Bit-exact with the reference packer (``quantize.py:95-152``,
    ``models/quantized.py:133-163``).
    """

    return _quantize(weight, group_size, 4)


def w8_quantize(weight: torch.Tensor, group_size: int = 64) -> tuple[torch.Tensor, torch.Tensor]:
    """Eight-bit pack: ``(int32 [out, in/4], bf16 scales [out, in/group])``.

    Bit-exact with ``quantize_int8`` (``quantize.py:155-172``) and
    ``pack_weight_int8`` (``models/quantized.py:166-172``).
    """

    return _quantize(weight, group_size, 8)


def quantize(weight: torch.Tensor, group_size: int = 64, bits: int = 4) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`w4_quantize` or :func:`w8_quantize` by width."""

    if bits not in CODES_PER_WORD:
        raise ValueError(f"bits must be 4 or 8, got {bits!r}")
    return _quantize(weight, group_size, bits)


def _dequantize(packed: torch.Tensor, scales: torch.Tensor, group_size: int, bits: int) -> torch.Tensor:
    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError("packed must be 2-D")
    rows, words = packed.shape
    inner = words * CODES_PER_WORD[bits]
    if group_size <= 0 or inner % group_size:
        raise ValueError(f"group size {group_size} does not divide {inner}")
    _expect(scales, "scales", BF16, (rows, inner // group_size))
    _ready(packed)
    out = torch.empty((rows, inner), dtype=BF16, device=packed.device)
    entry = _lib.library().aoto_hip_w4_dequantize if bits == 4 else _lib.library().aoto_hip_w8_dequantize
    _lib.check(entry(_ptr(packed), _ptr(scales), rows, inner, group_size, _ptr(out), _stream()))
    return out


def w4_dequantize(packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """``bf16(code * scale)`` ``[out, in]`` (``models/quantized.py:61-82``)."""

    return _dequantize(packed, scales, group_size, 4)


def w8_dequantize(packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """``bf16(code * scale)`` of an eight-bit pack (``models/quantized.py:84-107``)."""

    return _dequantize(packed, scales, group_size, 8)


def _gemv(
    bits: int,
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    norm_weight: torch.Tensor | None,
    eps: float,
    bias: torch.Tensor | None,
    alpha: float,
    beta: float,
    up: tuple[torch.Tensor, torch.Tensor] | None,
    out: torch.Tensor | None,
    lanes_per_row: int = 0,
) -> torch.Tensor:
    per_word = CODES_PER_WORD[bits]
    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError(f"packed must be 2-D [N, K/{per_word}]")
    n, words = packed.shape
    k = words * per_word
    if x.numel() != k:
        raise ValueError(f"x has {x.numel()} elements, the weight reduces over {k}")
    _expect(x, "x", BF16)
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(scales, "scales", BF16, (n, k // group_size))
    up_packed = up_scales = None
    if up is not None:
        up_packed, up_scales = up
        _expect(up_packed, "up packed", torch.int32, (n, words))
        _expect(up_scales, "up scales", BF16, (n, k // group_size))
    if norm_weight is not None:
        _expect(norm_weight, "norm_weight", BF16)
        if norm_weight.numel() != k:
            raise ValueError(f"norm_weight has {norm_weight.numel()} elements, expected {k}")
    if bias is not None:
        _expect(bias, "bias", BF16)
        if bias.numel() != n:
            raise ValueError(f"bias has {bias.numel()} elements, expected {n}")
    if out is None:
        out = torch.empty((n,), dtype=BF16, device=x.device)
    else:
        _expect(out, "out", BF16)
        if out.numel() != n:
            raise ValueError(f"out has {out.numel()} elements, expected {n}")
    _ready(x)
    lib = _lib.library()
    args = (_ptr(x), _ptr(packed), _ptr(scales), _ptr(up_packed), _ptr(up_scales), _ptr(norm_weight),
            float(eps), _ptr(bias), float(alpha), float(beta), _ptr(out), k, n, group_size)
    if bits == 4:
        _lib.check(lib.aoto_hip_w4_gemv(*args, int(lanes_per_row), _stream()))
    else:
        _lib.check(lib.aoto_hip_w8_gemv(*args, _stream()))
    return out


def w4_gemv(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    *,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    bias: torch.Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 1.0,
    up: tuple[torch.Tensor, torch.Tensor] | None = None,
    out: torch.Tensor | None = None,
    lanes_per_row: int = 0,
) -> torch.Tensor:
    """Decode GEMV ``y[N] = W4[N, K] @ x[K]`` with the fused prologue/epilogues.

    ``norm_weight``: RMSNorm prologue; ``bias``: addmm epilogue
    ``bf16(beta * bias + alpha * acc)``; ``up``: ``(packed, scales)`` of the up
    projection for the paired ``silu_mul`` epilogue (``packed`` is then gate).
    """

    return _gemv(4, x, packed, scales, group_size, norm_weight, eps, bias, alpha, beta, up, out, lanes_per_row)


def w8_gemv(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    *,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    bias: torch.Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 1.0,
    up: tuple[torch.Tensor, torch.Tensor] | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`w4_gemv` over an eight-bit pack ``int32 [N, K/4]``
    (``codegen/matmul.py:742-929``)."""

    return _gemv(8, x, packed, scales, group_size, norm_weight, eps, bias, alpha, beta, up, out)


def _i64(tensor: torch.Tensor, name: str) -> None:
    _expect(tensor, name, torch.int64)


def _matmul(
    bits: int,
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    bias: torch.Tensor | None,
    residual: torch.Tensor | None,
    gate: torch.Tensor | None,
    out: torch.Tensor | None,
    tile: int,
    splits: int,
    workspace: torch.Tensor | None,
) -> torch.Tensor:
    per_word = CODES_PER_WORD[bits]
    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError(f"packed must be 2-D [N, K/{per_word}]")
    n, words = packed.shape
    k = words * per_word
    _expect(x, "x", BF16)
    if x.shape[-1] != k:
        raise ValueError(f"x has last dimension {x.shape[-1]}, the weight reduces over {k}")
    m = x.numel() // k
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(scales, "scales", BF16, (n, k // group_size))
    for name, tensor, numel in (("bias", bias, n), ("residual", residual, m * n), ("gate", gate, m * n)):
        if tensor is not None:
            _expect(tensor, name, BF16)
            if tensor.numel() != numel:
                raise ValueError(f"{name} has {tensor.numel()} elements, expected {numel}")
    shape = tuple(x.shape[:-1]) + (n,)
    if out is None:
        out = torch.empty(shape, dtype=BF16, device=x.device)
    else:
        _expect(out, "out", BF16)
        if out.numel() != m * n:
            raise ValueError(f"out has {out.numel()} elements, expected {m * n}")
    _ready(x)
    _on_device(workspace)
    need = gemm_workspace_bytes(m, n, k, tile, splits)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty((need // 4,), dtype=torch.float32, device=x.device)
    entry = _lib.library().aoto_hip_w4_gemm if bits == 4 else _lib.library().aoto_hip_w8_gemm
    _lib.check(
        entry(
            _ptr(x), _ptr(packed), _ptr(scales), _ptr(bias), _ptr(residual), _ptr(gate), _ptr(out),
            m, n, k, group_size, int(tile), int(splits), _ptr(workspace if need else None), _stream(),
        )
    )
    return out


def w4_matmul(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    *,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    tile: int = 0,
    splits: int = 0,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Prefill W4 matmul ``[M, K] -> [M, N]`` on MFMA with one fused epilogue.

    ``bias`` ``[N]`` (q/k/v bias), ``residual`` ``[M, N]`` or ``gate`` ``[M, N]``
    (``silu_mul``: ``bf16(acc * silu(gate))``), as the reference's prefill GEMM.
    """

    return _matmul(4, x, packed, scales, group_size, bias, residual, gate, out, tile, splits, workspace)


def w8_matmul(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    *,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    tile: int = 0,
    splits: int = 0,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`w4_matmul` over an eight-bit pack ``int32 [N, K/4]``."""

    return _matmul(8, x, packed, scales, group_size, bias, residual, gate, out, tile, splits, workspace)


#: From this many rows (with K % 256 == 0) the prefill GEMMs' automatic plan
#: (tile = splits = 0) takes the wide-tile 32x32x16-MFMA kernel (the C ABI's kWideRows).
#: Where neither this rule nor :func:`lds_plan` applies, the C ABI picks among all instances
#: with a cost model (``modelled_plan`` in ``csrc/aoto_hip.cpp``).
WIDE_ROWS = 512


def wide_plan(m: int, n: int, k: int, *, paired: bool = False) -> tuple[int, int] | None:
    """The automatic plan's ``(tile, splits)`` for ``m`` rows of an ``[n, k]`` weight when
    it takes the wide kernel, else None: the Python mirror of the C ABI's
    ``wide_auto_plan`` (``csrc/aoto_hip.cpp``), for labels and host-side checks."""

    if m < WIDE_ROWS or k % 256:
        return None
    mb = (m + 127) // 128

    def blocks(bn):
        return -(-n // bn) * mb

    tile = 241
    if not paired and n % 384 == 0 and blocks(384) >= 224:
        tile = 243
    elif not paired and blocks(256) >= 224:
        tile = 441
    count = {243: blocks(384), 441: blocks(256), 241: blocks(128)}[tile]
    splits = -(-256 // count) if count < 160 else 1
    most = (k // 128) // 2
    splits = max(1, min(splits, most))
    # the launch cuts K into slices of whole 128-k steps: the count it actually runs
    steps = k // 128
    per = -(-steps // splits)
    return tile, -(-steps // per)


#: Tile codes of the dequant-once long-prefill kernel (``csrc/w4_gemm_lds.h``): the
#: single forms (256 x 128 and 256 x 192 blocks) and the paired gate/up form (256 x (64 + 64)).
LDS_TILE, LDS_WIDE_TILE, LDS_PAIRED_TILE = 822, 823, 821
#: the paired dequant-once forms for short prompts (128-row blocks of 4 waves):
#: 64 + 64 and 32 + 32 columns per block
LDS_SHORT_PAIRED_TILE, LDS_SHORT_NARROW_TILE = 812, 811
#: the single form's split-K partials for short prompts: 128 x 64 and 128 x 32 blocks
LDS_SPLIT_TILE, LDS_SPLIT_NARROW_TILE = 814, 813


def lds_plan(m: int, n: int, k: int, *, group_size: int = 64, paired: bool = False, bits: int = 4,
             gate: bool = False, rope: bool = False) -> int | None:
    """The tile code the automatic plan runs on the dequant-once kernel for this shape, else
    None: the Python mirror of the C ABI's ``lds_auto`` (4-bit codes, no gate epilogue,
    K % 64 == 0, a power-of-two group with an even count per row; from 1024 rows a grid
    of at least 256 blocks whose last round of 256 is at least 90% full: 128 columns per
    block where that fills the rounds, else 192; for a paired gate/up of 32-256 rows the
    128-row forms: 64 + 64 columns where that gives at least 128 blocks from 65 rows,
    else 32 + 32 where that fits 256 blocks; for a single projection of 32-256 rows with
    K >= 2048 and no RoPE epilogue (``rope``) the split-K form, 128 x 64 blocks where
    those give at least 64 column blocks, else 128 x 32)."""

    if bits != 4 or gate or k % 64 or group_size < 32 or group_size & (group_size - 1):
        return None
    if (k // group_size) % 2 or m * k * 2 >= 2 ** 31 or n * k // 2 >= 2 ** 31:
        return None
    if m < 1024:
        if m < 32 or m > 256:
            return None
        mb = -(-m // 128)
        if not paired:
            if rope or k < 2048:
                return None
            return LDS_SPLIT_TILE if -(-n // 64) * mb >= 64 else LDS_SPLIT_NARROW_TILE
        if m > 64 and -(-n // 64) * mb >= 128:
            return LDS_SHORT_PAIRED_TILE
        return LDS_SHORT_NARROW_TILE if -(-n // 32) * mb <= 256 else None
    def fills(bn):
        blocks = -(-n // bn) * -(-m // 256)
        rounds = -(-blocks // 256)
        return blocks >= 256 and blocks * 10 >= rounds * 256 * 9

    if paired:
        return LDS_PAIRED_TILE if fills(64) else None
    return LDS_TILE if fills(128) else LDS_WIDE_TILE if fills(192) else None


def gemm_workspace_bytes(m: int, n: int, k: int, tile: int = 0, splits: int = 0) -> int:
    """Workspace bytes :func:`w4_matmul` needs for this shape: split-K partials (0: no split)."""

    return int(_lib.library().aoto_hip_w4_gemm_workspace(int(m), int(n), int(k), int(tile), int(splits)))


def gate_up_workspace_bytes(m: int, n: int, k: int, tile: int = 0, splits: int = 0) -> int:
    """Workspace bytes :func:`w4_matmul_gate_up` needs (gate and up partials, 0: no split)."""

    return int(_lib.library().aoto_hip_w4_gemm_gate_up_workspace(int(m), int(n), int(k), int(tile), int(splits)))


def _matmul_gate_up(bits, x, gate_packed, gate_scales, up_packed, up_scales, group_size, out, tile, splits,
                    workspace):
    per_word = CODES_PER_WORD[bits]
    _expect(gate_packed, "gate_packed", torch.int32)
    if gate_packed.dim() != 2:
        raise ValueError(f"gate_packed must be 2-D [N, K/{per_word}]")
    n, words = gate_packed.shape
    k = words * per_word
    _expect(up_packed, "up_packed", torch.int32, (n, words))
    _expect(x, "x", BF16)
    if x.shape[-1] != k:
        raise ValueError(f"x has last dimension {x.shape[-1]}, the weights reduce over {k}")
    m = x.numel() // k
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(gate_scales, "gate_scales", BF16, (n, k // group_size))
    _expect(up_scales, "up_scales", BF16, (n, k // group_size))
    shape = tuple(x.shape[:-1]) + (n,)
    if out is None:
        out = torch.empty(shape, dtype=BF16, device=x.device)
    else:
        _expect(out, "out", BF16)
        if out.numel() != m * n:
            raise ValueError(f"out has {out.numel()} elements, expected {m * n}")
    _ready(x)
    _on_device(workspace)
    need = gate_up_workspace_bytes(m, n, k, tile, splits)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty((need // 4,), dtype=torch.float32, device=x.device)
    lib = _lib.library()
    entry = lib.aoto_hip_w4_gemm_gate_up if bits == 4 else lib.aoto_hip_w8_gemm_gate_up
    _lib.check(
        entry(
            _ptr(x), _ptr(gate_packed), _ptr(gate_scales), _ptr(up_packed), _ptr(up_scales), _ptr(out),
            m, n, k, group_size, int(tile), int(splits), _ptr(workspace if need else None), _stream(),
        )
    )
    return out


def w4_matmul_gate_up(x, gate_packed, gate_scales, up_packed, up_scales, group_size, *, out=None, tile=0,
                      splits=0, workspace=None):
    """Prefill MLP ``bf16(up(x) * silu(bf16(gate(x))))`` ``[M, K] -> [M, N]`` in one pass over x.

    The same values as ``w4_matmul(x, gate)`` followed by ``w4_matmul(x, up, gate=...)``
    (the reference's gate GEMM and silu_mul-epilogue up GEMM), up to the f32
    summation order of the split reduction.
    """

    return _matmul_gate_up(4, x, gate_packed, gate_scales, up_packed, up_scales, group_size, out, tile, splits,
                           workspace)


def w8_matmul_gate_up(x, gate_packed, gate_scales, up_packed, up_scales, group_size, *, out=None, tile=0,
                      splits=0, workspace=None):
    """:func:`w4_matmul_gate_up` over int8 packs (words ``[N, K/4]``)."""

    return _matmul_gate_up(8, x, gate_packed, gate_scales, up_packed, up_scales, group_size, out, tile, splits,
                           workspace)


def matmul_residual_norm(x, packed, scales, group_size, residual, norm_weight, eps, *, bits=4, out=None,
                         norm_out=None, tile=0, splits=0, workspace=None):
    """``y = bf16(x @ W^T + residual)`` then ``norm_out = rms_norm(y, norm_weight, eps)``.

    A decoder layer's o / down projection and the next block's RMSNorm: the same
    values as :func:`w4_matmul` (``residual=``) followed by :func:`rms_norm`, with the
    split-K sum and the norm in one launch. ``out`` may be ``residual`` (in place).
    Returns ``(y, norm_out)``.
    """

    per_word = CODES_PER_WORD[bits]
    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError(f"packed must be 2-D [N, K/{per_word}]")
    n, words = packed.shape
    k = words * per_word
    _expect(x, "x", BF16)
    if x.shape[-1] != k:
        raise ValueError(f"x has last dimension {x.shape[-1]}, the weight reduces over {k}")
    m = x.numel() // k
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(scales, "scales", BF16, (n, k // group_size))
    _expect(residual, "residual", BF16)
    _expect(norm_weight, "norm_weight", BF16, (n,))
    if residual.numel() != m * n:
        raise ValueError(f"residual has {residual.numel()} elements, expected {m * n}")
    shape = tuple(x.shape[:-1]) + (n,)
    out = torch.empty(shape, dtype=BF16, device=x.device) if out is None else out
    norm_out = torch.empty(shape, dtype=BF16, device=x.device) if norm_out is None else norm_out
    for name, t in (("out", out), ("norm_out", norm_out)):
        _expect(t, name, BF16)
        if t.numel() != m * n:
            raise ValueError(f"{name} has {t.numel()} elements, expected {m * n}")
    _ready(x)
    _on_device(workspace)
    need = gemm_workspace_bytes(m, n, k, tile, splits)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty((need // 4,), dtype=torch.float32, device=x.device)
    lib = _lib.library()
    entry = lib.aoto_hip_w4_gemm_residual_norm if bits == 4 else lib.aoto_hip_w8_gemm_residual_norm
    _lib.check(
        entry(
            _ptr(x), _ptr(packed), _ptr(scales), _ptr(residual), _ptr(out), m, n, k, group_size, int(tile),
            int(splits), _ptr(workspace if need else None), _ptr(norm_weight), float(eps), _ptr(norm_out),
            _stream(),
        )
    )
    return out, norm_out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """Row RMSNorm over the last dimension, ``bf16((x * rsqrt(mean(x^2) + eps)) * w)``."""

    _expect(x, "x", BF16)
    hidden = x.shape[-1]
    _expect(weight, "weight", BF16, (hidden,))
    rows = x.numel() // hidden
    if out is None:
        out = torch.empty_like(x)
    else:
        _expect(out, "out", BF16, tuple(x.shape))
    _ready(x)
    _lib.check(_lib.library().aoto_hip_rms_norm(_ptr(x), _ptr(weight), float(eps), _ptr(out), rows, hidden, _stream()))
    return out


def rope(
    x: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor
) -> torch.Tensor:
    """RoPE of ``x [B, H, S, D]`` with table rows ``positions [B, S]`` (int64)."""

    _expect(x, "x", BF16)
    if x.dim() != 4:
        raise ValueError("x must be [B, H, S, D]")
    batch, heads, seq, dim = x.shape
    _expect(cos_table, "cos_table", BF16)
    _expect(sin_table, "sin_table", BF16, tuple(cos_table.shape))
    if cos_table.shape[-1] != dim:
        raise ValueError("table width must equal the head dimension")
    _i64(positions, "positions")
    if positions.numel() != batch * seq:
        raise ValueError(f"positions must hold B*S = {batch * seq} entries")
    if batch != 1:
        raise ValueError("rope takes one batch row (positions are per token)")
    out = torch.empty_like(x)
    _ready(x)
    _lib.check(
        _lib.library().aoto_hip_rope(
            _ptr(x), _ptr(cos_table), _ptr(sin_table), _ptr(positions), 1, seq, _ptr(out),
            batch * heads * seq, dim, _stream(),
        )
    )
    return out


def rope_qkv_prefill(
    qkv: torch.Tensor,
    positions: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    pair: torch.Tensor,
    *,
    query_heads: int,
    kv_heads: int,
    head_dim: int,
    slot0: int,
    zero_prefix: bool = True,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Rotate q/k of ``qkv [B, M, W]`` into ``q [B, Hq, M, D]`` and fill ``pair [2, B, Hkv, cap, D]``."""

    _expect(qkv, "qkv", BF16)
    batch, tokens, width = qkv.shape
    if width != (query_heads + 2 * kv_heads) * head_dim:
        raise ValueError("qkv width does not match the head counts")
    _i64(positions, "positions")
    if positions.numel() != batch * tokens:
        raise ValueError("positions must be [B, M]")
    _expect(pair, "pair", BF16)
    if pair.dim() != 5 or tuple(pair.shape[:3]) != (2, batch, kv_heads) or pair.shape[4] != head_dim:
        raise ValueError(f"pair must be [2, {batch}, {kv_heads}, cap, {head_dim}], got {tuple(pair.shape)}")
    capacity = pair.shape[3]
    if q_out is None:
        q_out = torch.empty((batch, query_heads, tokens, head_dim), dtype=BF16, device=qkv.device)
    else:
        _expect(q_out, "q_out", BF16, (batch, query_heads, tokens, head_dim))
    _ready(qkv)
    _lib.check(
        _lib.library().aoto_hip_rope_qkv_prefill(
            _ptr(qkv), _ptr(positions), _ptr(cos_table), _ptr(sin_table), _ptr(q_out), _ptr(pair), batch,
            tokens, query_heads, kv_heads, head_dim, capacity, int(slot0), int(bool(zero_prefix)), _stream(),
        )
    )
    return q_out


def matmul_qkv_rope(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    positions: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    pair: torch.Tensor,
    *,
    query_heads: int,
    kv_heads: int,
    head_dim: int,
    slot0: int,
    bias: torch.Tensor | None = None,
    zero_prefix: bool = True,
    bits: int = 4,
    out: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
    tile: int = 0,
    splits: int = 0,
    workspace: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The packed q/k/v projection ``out = bf16(x @ W^T + bias)`` ``[M, W]`` with RoPE of q into
    ``q_out [1, Hq, M, D]`` and the rotated keys / values into ``pair [2, 1, Hkv, cap, D]`` at
    ``slot0``: :func:`w4_matmul` then :func:`rope_qkv_prefill` (batch 1) in one launch - RoPE in
    the GEMM's epilogue when unsplit (``splits=0`` prefers it whenever a block's columns are
    whole heads), in the split-K sum's launch when split. Returns ``(out, q_out)``."""

    per_word = CODES_PER_WORD[bits]
    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError(f"packed must be 2-D [N, K/{per_word}]")
    n, words = packed.shape
    k = words * per_word
    if n != (query_heads + 2 * kv_heads) * head_dim:
        raise ValueError("the projection's rows do not match the head counts")
    _expect(x, "x", BF16)
    if x.shape[-1] != k:
        raise ValueError(f"x has last dimension {x.shape[-1]}, the weight reduces over {k}")
    m = x.numel() // k
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(scales, "scales", BF16, (n, k // group_size))
    if bias is not None:
        _expect(bias, "bias", BF16, (n,))
    _i64(positions, "positions")
    if positions.numel() != m:
        raise ValueError("positions must hold one entry per row of x")
    _expect(pair, "pair", BF16)
    if pair.dim() != 5 or tuple(pair.shape[:3]) != (2, 1, kv_heads) or pair.shape[4] != head_dim \
            or not pair.is_contiguous():
        raise ValueError(f"pair must be a contiguous [2, 1, {kv_heads}, cap, {head_dim}], got {tuple(pair.shape)}")
    capacity = pair.shape[3]
    if out is None:
        out = torch.empty((m, n), dtype=BF16, device=x.device)
    elif out.numel() != m * n:
        raise ValueError(f"out has {out.numel()} elements, expected {m * n}")
    if q_out is None:
        q_out = torch.empty((1, query_heads, m, head_dim), dtype=BF16, device=x.device)
    else:
        _expect(q_out, "q_out", BF16, (1, query_heads, m, head_dim))
    _ready(x)
    lib = _lib.library()
    _on_device(workspace)
    need = int(lib.aoto_hip_w4_gemm_qkv_rope_workspace(m, k, int(tile), int(splits), query_heads, kv_heads, head_dim))
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty((need // 4,), dtype=torch.float32, device=x.device)
    entry = lib.aoto_hip_w4_gemm_qkv_rope if bits == 4 else lib.aoto_hip_w8_gemm_qkv_rope
    _lib.check(
        entry(
            _ptr(x), _ptr(packed), _ptr(scales), _ptr(bias), _ptr(out), m, k, group_size, int(tile), int(splits),
            _ptr(workspace if need else None), _ptr(positions), _ptr(cos_table), _ptr(sin_table), _ptr(q_out),
            _ptr(pair), query_heads, kv_heads, head_dim, capacity, int(slot0), int(bool(zero_prefix)), _stream(),
        )
    )
    return out, q_out


def rope_kv_cache_append(
    row: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    position: int,
    pair_out: torch.Tensor,
    *,
    pair_in: torch.Tensor | None,
    query_heads: int,
    query_start: int,
    key_start: int,
    value_start: int,
    ring_slot: int | None = None,
    step_state: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The decode ``rope_kv_cache_append``: returns ``q [B, Hq, D]``.

    ``pair_in`` given: the reference's roll into ``pair_out``. ``ring_slot``
    given instead: the new key/value is written in place at that slot.
    """

    _expect(row, "row", BF16)
    batch, width = row.shape[0], row.shape[-1]
    _expect(pair_out, "pair_out", BF16)
    _, b2, kv_heads, capacity, head_dim = pair_out.shape
    if b2 != batch:
        raise ValueError("row and pair batch differ")
    mode = 1 if (ring_slot is not None or step_state is not None) else 0
    if mode == 0:
        if pair_in is None:
            raise ValueError("the roll needs pair_in")
        _expect(pair_in, "pair_in", BF16, tuple(pair_out.shape))
    if q_out is None:
        q_out = torch.empty((batch, query_heads, head_dim), dtype=BF16, device=row.device)
    _ready(row)
    _lib.check(
        _lib.library().aoto_hip_rope_kv_cache_append(
            _ptr(row), width, _ptr(cos_table), _ptr(sin_table), int(position), _ptr(pair_in), _ptr(pair_out),
            _ptr(q_out), batch, query_heads, kv_heads, capacity, head_dim, query_start, key_start, value_start,
            mode, int(ring_slot or 0), _ptr(step_state), _stream(),
        )
    )
    return q_out


def decode_attention_workspace(batch: int, query_heads: int, kv_heads: int, capacity: int, head_dim: int,
                               splits: int = 0, device=None) -> torch.Tensor:
    """A workspace for the split-K records of :func:`decode_attention` with these shapes (on ``device``; a GPU's, and
    torch's default device is the host unless a program sets it)."""

    size = _lib.library().aoto_hip_decode_attention_workspace(batch, query_heads, kv_heads, capacity, head_dim, splits)
    return torch.zeros((max(size, 16),), dtype=torch.uint8, device=device)


def decode_attention(
    q: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    *,
    valid: int | None = None,
    ring_offset: int = 0,
    mask: torch.Tensor | None = None,
    scale: float | None = None,
    workspace: torch.Tensor | None = None,
    splits: int = 0,
    step_state: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Single-query GQA attention: ``q [B, Hq, D]`` over ``keys/values [B, Hkv, cap, D]``."""

    _expect(q, "q", BF16)
    batch, query_heads, head_dim = q.shape
    if keys.dtype != BF16 or values.dtype != BF16 or keys.shape != values.shape or keys.dim() != 4:
        raise ValueError("keys/values must be bf16 [B, Hkv, cap, D] of one shape")
    if keys.stride(-1) != 1 or keys.stride(-2) != head_dim or values.stride() != keys.stride():
        raise ValueError("keys/values rows must be contiguous with matching strides")
    _, kv_heads, capacity, _ = keys.shape
    if scale is None:
        scale = ctypes.c_float(head_dim ** -0.5).value
    mask_ptr = None
    mask_stride = 0
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError("mask must be bool")
        mask = mask.reshape(-1, capacity).to(torch.uint8).contiguous()
        mask_stride = capacity if mask.shape[0] == batch else 0
        mask_ptr = mask
    elif valid is None and step_state is None:
        raise ValueError("pass valid=, mask= or step_state=")
    if out is None:
        out = torch.empty_like(q)
    _on_device(workspace)
    _ready(q)
    _lib.check(
        _lib.library().aoto_hip_decode_attention(
            _ptr(q), _ptr(keys), _ptr(values), keys.stride(0), keys.stride(1), _ptr(mask_ptr), mask_stride,
            int(valid or 0), int(ring_offset), batch, query_heads, kv_heads, capacity, head_dim, float(scale),
            int(splits), _ptr(workspace), _ptr(step_state), _ptr(out), _stream(),
        )
    )
    return out


def decode_rope_attention(
    row: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    pair: torch.Tensor,
    *,
    query_heads: int,
    query_start: int,
    key_start: int,
    value_start: int,
    position: int = 0,
    slot: int = 0,
    valid: int = 0,
    ring_offset: int = 0,
    step_state: torch.Tensor | None = None,
    scale: float | None = None,
    workspace: torch.Tensor | None = None,
    splits: int = 0,
    rope_rows: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """RoPE + in-place KV write at ``slot`` + single-query attention over ``pair [2, B, Hkv, cap, D]``.

    ``rope_rows`` (bf16 ``[2, D]``: cos row, sin row of the current position) replaces the table lookup.
    """

    _expect(row, "row", BF16)
    _expect(pair, "pair", BF16)
    _, batch, kv_heads, capacity, head_dim = pair.shape
    width = row.shape[-1]
    if row.numel() != batch * width:
        raise ValueError("row must be [B, W]")
    if scale is None:
        scale = ctypes.c_float(head_dim ** -0.5).value
    if out is None:
        out = torch.empty((batch, query_heads, head_dim), dtype=BF16, device=row.device)
    if rope_rows is not None:
        _expect(rope_rows, "rope_rows", BF16, (2, head_dim))
    keys, values = pair[0], pair[1]
    _on_device(workspace)
    _ready(row)
    _lib.check(
        _lib.library().aoto_hip_decode_rope_attention(
            _ptr(row), width, query_start, key_start, value_start, _ptr(cos_table), _ptr(sin_table), _ptr(keys),
            _ptr(values), keys.stride(0), keys.stride(1), int(position), int(slot), int(valid), int(ring_offset),
            batch, query_heads, kv_heads, capacity, head_dim, float(scale), int(splits), _ptr(workspace),
            _ptr(step_state), _ptr(rope_rows), _ptr(out), _stream(),
        )
    )
    return out


def prefill_attention(
    q: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    *,
    causal: bool = True,
    key_start: int = 0,
    mask: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Prefill GQA attention: ``q [B, Hq, M, D]``, ``keys/values [B, Hkv, Mk, D]`` (rows contiguous)
    -> ``[B, M, Hq*D]``."""

    _expect(q, "q", BF16)
    batch, query_heads, tokens, head_dim = q.shape
    if keys.dtype != BF16 or values.dtype != BF16 or keys.shape != values.shape or keys.dim() != 4:
        raise ValueError("keys/values must be bf16 [B, Hkv, Mk, D] of one shape")
    if keys.stride(-1) != 1 or keys.stride(-2) != head_dim or values.stride() != keys.stride():
        raise ValueError("keys/values rows must be contiguous with matching strides")
    _, kv_heads, key_tokens, _ = keys.shape
    if scale is None:
        scale = ctypes.c_float(head_dim ** -0.5).value
    mask_ptr = None
    mask_stride = 0
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError("mask must be bool")
        mask = mask.reshape(-1, tokens, key_tokens).to(torch.uint8).contiguous()
        mask_stride = tokens * key_tokens if mask.shape[0] == batch and batch > 1 else 0
        mask_ptr = mask
    if out is None:
        out = torch.empty((batch, tokens, query_heads * head_dim), dtype=BF16, device=q.device)
    _ready(q)
    _lib.check(
        _lib.library().aoto_hip_prefill_attention(
            _ptr(q), _ptr(keys), _ptr(values), keys.stride(0), keys.stride(1), _ptr(mask_ptr), mask_stride,
            int(bool(causal)), int(key_start), batch, tokens, key_tokens, query_heads, kv_heads, head_dim,
            float(scale), _ptr(out), _stream(),
        )
    )
    return out


def embedding(weight: torch.Tensor, ids: torch.Tensor, *, out: torch.Tensor | None = None,
              error: torch.Tensor | None = None) -> torch.Tensor:
    """``weight[ids]`` for int64 device ``ids``; out-of-range ids give zero rows and set ``error``."""

    _expect(weight, "weight", BF16)
    _i64(ids, "ids")
    vocab, hidden = weight.shape
    count = ids.numel()
    if out is None:
        out = torch.empty(tuple(ids.shape) + (hidden,), dtype=BF16, device=weight.device)
    if error is not None:
        _expect(error, "error", torch.int32)
    _ready(weight)
    _lib.check(
        _lib.library().aoto_hip_embedding(
            _ptr(weight), _ptr(ids), count, hidden, vocab, _ptr(out), _ptr(error), _stream()
        )
    )
    return out


def argmax(logits: torch.Tensor, *, out: torch.Tensor | None = None, history: torch.Tensor | None = None,
           history_len: torch.Tensor | None = None) -> torch.Tensor:
    """First-index argmax over the last dimension of bf16 ``logits`` -> int64 ``[rows]``."""

    _expect(logits, "logits", BF16)
    n = logits.shape[-1]
    rows = logits.numel() // n
    if out is None:
        out = torch.empty((rows,), dtype=torch.int64, device=logits.device)
    _ready(logits)
    _lib.check(
        _lib.library().aoto_hip_argmax(
            _ptr(logits), rows, n, n, _ptr(out), _ptr(history), _ptr(history_len), _stream()
        )
    )
    return out


def argmax_key_count(k: int, n: int, group_size: int) -> int:
    """Keys ``w4_gemv_argmax`` writes for a ``[n, k]`` weight; 0 when the fused form does not take the shape."""

    return int(_lib.library().aoto_hip_w4_gemv_argmax_keys(int(k), int(n), int(group_size)))


def w4_gemv_argmax(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    keys: torch.Tensor,
    *,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """LM-head GEMV (optional RMSNorm prologue) that also writes greedy-argmax keys for ``argmax_finish``.

    ``keys`` is an int64 device buffer of at least ``argmax_key_count(K, N, group)`` entries.
    Returns the bf16 logits ``[N]`` (identical to ``w4_gemv``'s).
    """

    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError("packed must be 2-D [N, K/8]")
    n, words = packed.shape
    k = words * 8
    _expect(x, "x", BF16)
    if x.numel() != k:
        raise ValueError(f"x has {x.numel()} elements, the weight reduces over {k}")
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(scales, "scales", BF16, (n, k // group_size))
    _i64(keys, "keys")
    if norm_weight is not None:
        _expect(norm_weight, "norm_weight", BF16)
        if norm_weight.numel() != k:
            raise ValueError(f"norm_weight has {norm_weight.numel()} elements, expected {k}")
    if out is None:
        out = torch.empty((n,), dtype=BF16, device=x.device)
    else:
        _expect(out, "out", BF16)
        if out.numel() != n:
            raise ValueError(f"out has {out.numel()} elements, expected {n}")
    _ready(x)
    _lib.check(
        _lib.library().aoto_hip_w4_gemv_argmax(
            _ptr(x), _ptr(packed), _ptr(scales), _ptr(norm_weight), float(eps), _ptr(out), k, n, group_size,
            _ptr(keys), keys.numel(), _stream(),
        )
    )
    return out


def argmax_finish(
    keys: torch.Tensor,
    count: int,
    *,
    out: torch.Tensor,
    history: torch.Tensor | None = None,
    history_len: torch.Tensor | None = None,
    step_state: torch.Tensor | None = None,
    capacity: int = 0,
    embedding: torch.Tensor | None = None,
    hidden_out: torch.Tensor | None = None,
    error: torch.Tensor | None = None,
    rope_tables: tuple[torch.Tensor, torch.Tensor] | None = None,
    rope_rows: torch.Tensor | None = None,
) -> torch.Tensor:
    """Reduce ``count`` argmax keys to the greedy token ``out[0]``; optionally append it to ``history``,
    advance ``step_state``, gather its ``embedding`` row into ``hidden_out`` and copy the advanced
    position's rows of ``rope_tables`` (cos, sin ``[capacity, D]``) into ``rope_rows`` ``[2, D]``."""

    _i64(keys, "keys")
    _i64(out, "out")
    if not 0 < count <= keys.numel():
        raise ValueError(f"count {count} is outside (0, {keys.numel()}]")
    if step_state is not None:
        _expect(step_state, "step_state", torch.int32, (4,))
    hidden = rows = 0
    if embedding is not None:
        _expect(embedding, "embedding", BF16)
        rows, hidden = embedding.shape
        if hidden_out is None or hidden_out.numel() != hidden:
            raise ValueError("hidden_out must hold one embedding row")
        _expect(hidden_out, "hidden_out", BF16)
    if error is not None:
        _expect(error, "error", torch.int32)
    cos_table = sin_table = None
    head_dim = 0
    if rope_rows is not None:
        if rope_tables is None or step_state is None:
            raise ValueError("rope_rows needs rope_tables and step_state")
        cos_table, sin_table = rope_tables
        head_dim = cos_table.shape[-1]
        _expect(cos_table, "cos table", BF16, (int(capacity), head_dim))
        _expect(sin_table, "sin table", BF16, (int(capacity), head_dim))
        _expect(rope_rows, "rope_rows", BF16, (2, head_dim))
    _ready(keys)
    _lib.check(
        _lib.library().aoto_hip_argmax_finish(
            _ptr(keys), int(count), _ptr(out), _ptr(history), _ptr(history_len), _ptr(step_state), int(capacity),
            _ptr(embedding), int(rows), int(hidden), _ptr(hidden_out), _ptr(error), _ptr(cos_table),
            _ptr(sin_table), int(head_dim), _ptr(rope_rows), _stream(),
        )
    )
    return out


def gemv_finish_supported(k: int, n: int, group_size: int, key_count: int) -> bool:
    """Whether ``w4_gemv_finish`` takes a ``[n, k]`` weight and ``key_count`` keys (a shape check, no launch)."""

    if not 0 < key_count <= int(_lib.library().aoto_hip_w4_gemv_finish_max_keys()):
        return False
    if group_size < 32 or group_size & (group_size - 1) or k % group_size or (k // group_size) % 2:
        return False
    return (k == 896 and n <= 8192) or (k == 4096 and n <= 16384)


def w4_gemv_finish(
    keys: torch.Tensor,
    count: int,
    embedding: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    group_size: int,
    *,
    norm_weight: torch.Tensor,
    eps: float,
    out: torch.Tensor,
    token_out: torch.Tensor,
    hidden_out: torch.Tensor,
    bias: torch.Tensor | None = None,
    history: torch.Tensor | None = None,
    history_len: torch.Tensor | None = None,
    step_state: torch.Tensor | None = None,
    capacity: int = 0,
    error: torch.Tensor | None = None,
    rope_tables: tuple[torch.Tensor, torch.Tensor] | None = None,
    rope_rows: torch.Tensor | None = None,
) -> torch.Tensor:
    """``argmax_finish`` of ``count`` keys folded into the next step's first W4 GEMV.

    The greedy token's ``embedding`` row is the GEMV's x (RMSNorm prologue with
    ``norm_weight``, optional ``bias``): ``out`` [N] equals ``w4_gemv`` of that row.
    The token, history, step state, RoPE rows and the raw row (into ``hidden_out``)
    are recorded as ``argmax_finish`` records them.
    """

    _i64(keys, "keys")
    _i64(token_out, "token_out")
    _expect(packed, "packed", torch.int32)
    if packed.dim() != 2:
        raise ValueError("packed must be 2-D [N, K/8]")
    n, words = packed.shape
    k = words * 8
    _expect(embedding, "embedding", BF16)
    rows, hidden = embedding.shape
    if hidden != k:
        raise ValueError(f"embedding rows have {hidden} elements, the weight reduces over {k}")
    if group_size <= 0 or k % group_size:
        raise ValueError(f"group size {group_size} does not divide K={k}")
    _expect(scales, "scales", BF16, (n, k // group_size))
    _expect(norm_weight, "norm_weight", BF16)
    if norm_weight.numel() != k:
        raise ValueError(f"norm_weight has {norm_weight.numel()} elements, expected {k}")
    if bias is not None:
        _expect(bias, "bias", BF16)
        if bias.numel() != n:
            raise ValueError(f"bias has {bias.numel()} elements, expected {n}")
    _expect(out, "out", BF16)
    if out.numel() != n:
        raise ValueError(f"out has {out.numel()} elements, expected {n}")
    _expect(hidden_out, "hidden_out", BF16)
    if hidden_out.numel() != k:
        raise ValueError("hidden_out must hold one embedding row")
    if not 0 < count <= keys.numel():
        raise ValueError(f"count {count} is outside (0, {keys.numel()}]")
    if step_state is not None:
        _expect(step_state, "step_state", torch.int32, (4,))
    if error is not None:
        _expect(error, "error", torch.int32)
    cos_table = sin_table = None
    head_dim = 0
    if rope_rows is not None:
        if rope_tables is None or step_state is None:
            raise ValueError("rope_rows needs rope_tables and step_state")
        cos_table, sin_table = rope_tables
        head_dim = cos_table.shape[-1]
        _expect(cos_table, "cos table", BF16, (int(capacity), head_dim))
        _expect(sin_table, "sin table", BF16, (int(capacity), head_dim))
        _expect(rope_rows, "rope_rows", BF16, (2, head_dim))
    _ready(keys)
    _lib.check(
        _lib.library().aoto_hip_w4_gemv_finish(
            _ptr(keys), int(count), _ptr(embedding), int(rows), _ptr(packed), _ptr(scales), _ptr(norm_weight),
            float(eps), _ptr(bias), 1.0, 1.0, _ptr(out), k, n, int(group_size), _ptr(token_out), _ptr(history),
            _ptr(history_len), _ptr(step_state), int(capacity), _ptr(cos_table), _ptr(sin_table), int(head_dim),
            _ptr(rope_rows), _ptr(hidden_out), _ptr(error), _stream(),
        )
    )
    return out


def step_advance(step_state: torch.Tensor, capacity: int) -> None:
    """Advance the int32 device step state ``{position, valid, ring_offset, slot}`` by one token."""

    _expect(step_state, "step_state", torch.int32, (4,))
    _ready(step_state)
    _lib.check(_lib.library().aoto_hip_step_advance(_ptr(step_state), int(capacity), _stream()))


# ------------------------------------------------------------------------------------------------------------------
# Requests of different lengths over one paged key/value cache: a step's bookkeeping, the cache write, the attention
# and the verification of drafted tokens. A layer's cache is a pair ``keys, values`` of bf16 ``[pages, Hkv, page, D]``
# tensors (views with rows of ``D`` contiguous elements will do, a ``[pages, page, Hkv, D]`` cache transposed for one);
# slot ``s`` is row ``s % page`` of page ``s // page``.

#: Bits raised in the ``error`` tensor of the paged operators (``AOTO_PAGED_*`` in ``include/aoto_hip.h``).
PAGED_TOKENS_CUT, PAGED_NO_PAGES, PAGED_TABLE_FULL, PAGED_BAD_SLOT, PAGED_BAD_POSITION = 1, 2, 4, 8, 16


class PagedStep(NamedTuple):
    """What :func:`paged_tables` says of a step (``block_tables`` are extended in place)."""

    query_start: torch.Tensor   # int32 [R + 1]: the rows of request r are query_start[r] .. query_start[r + 1]
    kv_lens: torch.Tensor       # int32 [R]: cached tokens with the step's own
    positions: torch.Tensor     # int64 [max_tokens]
    slots: torch.Tensor         # int64 [max_tokens], -1 behind the last token
    page_counts: torch.Tensor   # int32 [R]
    free_start: torch.Tensor    # int32 [1]


def _on_current(name: str, tensor: torch.Tensor) -> int:
    """The device of ``tensor``, the current one: the launch goes to its stream, and a tensor of another device would
    be read across the link, or not at all."""

    device = tensor.get_device()
    if device != torch.cuda.current_device():
        raise ValueError(f"{name} is on {tensor.device}, the current device is cuda:{torch.cuda.current_device()}")
    return device


def _expect_all(device: int, tensors) -> None:
    """:func:`_expect` for ``(tensor, name, dtype, shape)`` of one call, all of them on ``device``."""

    for tensor, name, dtype, shape in tensors:
        if not (isinstance(tensor, torch.Tensor) and tensor.get_device() == device and tensor.dtype is dtype
                and tensor.is_contiguous() and (shape is None or tensor.shape == shape)):
            _expect(tensor, name, dtype, shape)
            raise ValueError(f"{name} is on {tensor.device}, the call's other tensors on cuda:{device}")


def _expect_rows(tensor: torch.Tensor, name: str, dtype: torch.dtype, dims: int, device: int) -> None:
    """A ``dims``-dimensional operand whose rows (last dimension) are contiguous, at any other strides."""

    if (isinstance(tensor, torch.Tensor) and tensor.is_cuda and tensor.get_device() == device
            and tensor.dtype is dtype and tensor.dim() == dims and tensor.stride(-1) == 1):
        return
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(tensor).__name__}")
    if tensor.device.type != "cuda":
        raise ValueError(f"{name} must be on the GPU, got {tensor.device}")
    if tensor.get_device() != device:
        raise ValueError(f"{name} is on {tensor.device}, the call's other tensors on cuda:{device}")
    if tensor.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {tensor.dtype}")
    if tensor.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(tensor.shape)}")
    if tensor.shape[-1] != 1 and tensor.stride(-1) != 1 and tensor.numel():
        raise ValueError(f"{name}'s rows must be contiguous")


def _expect_pages(keys: torch.Tensor, values: torch.Tensor, device: int) -> tuple[tuple, tuple]:
    """``(pages, Hkv, page, D)`` of a layer's cache, and its strides."""

    _expect_rows(keys, "keys", BF16, 4, device)
    _expect_rows(values, "values", BF16, 4, device)
    shape, strides = keys.shape, keys.stride()
    if shape != values.shape or strides != values.stride():
        raise ValueError("keys and values must have one shape and the same strides")
    return shape, strides


def paged_tables(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    page_counts: torch.Tensor,
    free_pages: torch.Tensor,
    free_start: torch.Tensor,
    *,
    page_size: int,
    max_tokens: int,
    shares: torch.Tensor | None = None,
    step: PagedStep | None = None,
    error: torch.Tensor | None = None,
) -> PagedStep:
    """A step's pages, block tables and token maps, built on the GPU from the requests' lengths.

    Request ``r`` has ``context_lens[r]`` cached tokens and gets ``new_lens[r]`` (int32 ``[R]``). Where the
    ``page_counts[r]`` pages of its row of ``block_tables`` (int32 ``[R, max_blocks]``) do not hold them all, the next
    pages of ``free_pages[free_start:]`` (int32) are entered there, requests in order; a request keeps pages that it
    does not need yet (drafted tokens that did not stand leave some). Token ``i`` of request ``r`` is row
    ``query_start[r] + i`` of the step, at position ``context_lens[r] + i``, in slot
    ``block_tables[r][position // page_size] * page_size + position % page_size``; rows from the last token to
    ``max_tokens`` have position 0 and slot -1.

    ``step`` gives the tensors to write (a captured step replays into them); its ``page_counts`` and ``free_start``
    may be the ones passed in. ``error`` (int32 ``[1]``) collects ``PAGED_TOKENS_CUT`` (more tokens than
    ``max_tokens``: the last are left out), ``PAGED_NO_PAGES`` (the free list ran out: table entries and slots of -1)
    and ``PAGED_TABLE_FULL`` (a request longer than its row: slots of -1). With ``shares`` (int32 ``[pages]``, where
    rows go on from others by :func:`paged_fork`) also ``PAGED_ROW_SHARED``: a token's page is held by others too, whom
    it would be written over (slots of -1).
    """

    _expect(context_lens, "context_lens", torch.int32)
    device = _on_current("context_lens", context_lens)
    requests = context_lens.numel()
    max_tokens = int(max_tokens)
    if context_lens.dim() != 1:
        raise ValueError(f"context_lens must be [R], got {tuple(context_lens.shape)}")
    _expect_all(device, (
        (new_lens, "new_lens", torch.int32, (requests,)), (page_counts, "page_counts", torch.int32, (requests,)),
        (free_pages, "free_pages", torch.int32, None), (free_start, "free_start", torch.int32, (1,)),
    ))
    _expect_rows(block_tables, "block_tables", torch.int32, 2, device)
    if block_tables.shape[0] != requests:
        raise ValueError(f"block_tables must have {requests} rows, got {block_tables.shape[0]}")
    if error is not None:
        _expect_all(device, ((error, "error", torch.int32, (1,)),))
    if shares is not None:
        _expect_all(device, ((shares, "shares", torch.int32, None),))
        if shares.dim() != 1 or not shares.numel():
            raise ValueError(f"shares must be [pages], got {tuple(shares.shape)}")
    if max_tokens < 0:
        raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
    if step is None:
        lens = context_lens.new_empty((3 * requests + 2,))
        start, kv, counts, first = lens.split_with_sizes((requests + 1, requests, requests, 1))
        maps = torch.empty((2, max_tokens), dtype=torch.int64, device=context_lens.device)
        step = PagedStep(start, kv, *maps.unbind(), counts, first)
    else:
        _expect_all(device, (
            (step.query_start, "step.query_start", torch.int32, (requests + 1,)),
            (step.kv_lens, "step.kv_lens", torch.int32, (requests,)),
            (step.positions, "step.positions", torch.int64, (max_tokens,)),
            (step.slots, "step.slots", torch.int64, (max_tokens,)),
            (step.page_counts, "step.page_counts", torch.int32, (requests,)),
            (step.free_start, "step.free_start", torch.int32, (1,)),
        ))
    _ready(context_lens)
    _lib.check(
        _lib.library().aoto_hip_paged_tables_shared(
            _ptr(context_lens), _ptr(new_lens), _ptr(block_tables), block_tables.stride(0), _ptr(page_counts),
            _ptr(free_pages), _ptr(free_start), _ptr(shares), requests, block_tables.shape[1], free_pages.numel(),
            0 if shares is None else shares.numel(), int(page_size), max_tokens, _ptr(step.query_start),
            _ptr(step.kv_lens), _ptr(step.positions), _ptr(step.slots), _ptr(step.page_counts), _ptr(step.free_start),
            _ptr(error), _stream(device),
        )
    )
    return step


def paged_rope_append(
    qkv: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    *,
    query_heads: int,
    q_out: torch.Tensor | None = None,
    error: torch.Tensor | None = None,
) -> torch.Tensor:
    """RoPE of a step's ``qkv [T, (Hq + 2 Hkv) D]`` rows and the write of one layer's cache: returns ``q [T, Hq, D]``.

    Row ``t`` is rotated by row ``positions[t]`` of the tables (bf16 ``[P, D]``), its key and value go to slot
    ``slots[t]`` of ``keys``, ``values`` (int64 ``[T]`` both). A row of slot -1 (behind the step's last token) writes
    nothing, its query included; so does one whose slot or position is out of range, which raises ``PAGED_BAD_SLOT``
    or ``PAGED_BAD_POSITION`` in ``error`` (int32 ``[1]``). Slots other than -1 must not repeat within a call.
    """

    _expect_rows(qkv, "qkv", BF16, 2, qkv.get_device() if isinstance(qkv, torch.Tensor) else 0)
    device = _on_current("qkv", qkv)
    (pages, kv_heads, page, dim), (page_stride, head_stride, slot_stride, _) = _expect_pages(keys, values, device)
    tokens, width = qkv.shape
    query_heads = int(query_heads)
    if query_heads <= 0 or width != (query_heads + 2 * kv_heads) * dim:
        raise ValueError(f"qkv rows of {width} do not hold {query_heads} + 2 x {kv_heads} heads of {dim}")
    _expect_all(device, ((positions, "positions", torch.int64, (tokens,)), (slots, "slots", torch.int64, (tokens,)),
                         (cos_table, "cos_table", BF16, None)))
    if cos_table.dim() != 2 or cos_table.shape[1] != dim:
        raise ValueError(f"cos_table must be [P, {dim}], got {tuple(cos_table.shape)}")
    _expect_all(device, ((sin_table, "sin_table", BF16, cos_table.shape),))
    if error is not None:
        _expect_all(device, ((error, "error", torch.int32, (1,)),))
    if q_out is None:
        q_out = qkv.new_empty((tokens, query_heads, dim))
    else:
        _expect_all(device, ((q_out, "q_out", BF16, (tokens, query_heads, dim)),))
    _ready(qkv)
    _lib.check(
        _lib.library().aoto_hip_paged_rope_append(
            _ptr(qkv), qkv.stride(0), _ptr(positions), _ptr(slots), _ptr(cos_table), _ptr(sin_table),
            cos_table.shape[0], _ptr(keys), _ptr(values), page_stride, head_stride, slot_stride, pages, page, tokens,
            query_heads, kv_heads, dim, _ptr(q_out), _ptr(error), _stream(device),
        )
    )
    return q_out


def paged_attention_workspace(tokens: int, requests: int, max_blocks: int, page_size: int, query_heads: int,
                              kv_heads: int, head_dim: int, *, max_query_len: int = 0, max_kv_len: int = 0,
                              device=None) -> torch.Tensor:
    """A workspace for :func:`paged_attention` with these shapes and bounds (on ``device``; a GPU's, and torch's
    default device is the host unless a program sets it)."""

    size = _lib.library().aoto_hip_paged_attention_workspace(
        int(tokens), int(requests), int(max_blocks), int(page_size), int(query_heads), int(kv_heads), int(head_dim),
        int(max_query_len), int(max_kv_len))
    return torch.empty((max(size, 16),), dtype=torch.uint8, device=device)


def paged_attention(
    q: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    block_tables: torch.Tensor,
    query_start: torch.Tensor,
    kv_lens: torch.Tensor,
    *,
    causal: bool = True,
    scale: float | None = None,
    max_query_len: int = 0,
    max_kv_len: int = 0,
    workspace: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """GQA attention of the requests' new tokens ``q [T, Hq, D]`` over their pages -> ``[T, Hq * D]``.

    Request ``r`` has the rows ``query_start[r] .. query_start[r + 1]`` (int32 ``[R + 1]``) and ``kv_lens[r]`` keys
    (int32 ``[R]``), its own new ones among them, in the pages that ``block_tables[r]`` (int32 ``[R, max_blocks]``)
    names: one token, a few drafted ones or a chunk of a prompt, side by side. Row ``i`` of ``n`` sees the keys up to
    its own, ``j <= kv_lens[r] - n + i`` (all of them with ``causal=False``); keys past the block table row or in
    entries that name no page are not there, and a row that sees none gives 0. NaN and infinities in what a row sees
    are the softmax's: a NaN or +inf among its scores, or none but -inf, makes it NaN, a value is in its dim however
    small the weight. Rows before ``query_start[0]`` and from ``query_start[R]`` on keep what ``out`` held. The lengths
    are read on the GPU; ``max_query_len`` and ``max_kv_len`` (0: not known) are the caller's bounds on a request's
    rows and keys, which choose the launch, and with it the order of sums and whether weights are rounded to bf16 or
    kept to 16 bits; what is computed goes by the lengths. ``workspace`` (:func:`paged_attention_workspace`; allocated
    where it is missing or too small) is written by the call: calls that share one are ordered on one stream.
    """

    _expect_rows(q, "q", BF16, 3, q.get_device() if isinstance(q, torch.Tensor) else 0)
    device = _on_current("q", q)
    tokens, query_heads, dim = q.shape
    (pages, kv_heads, page, key_dim), (page_stride, head_stride, slot_stride, _) = _expect_pages(keys, values, device)
    if key_dim != dim:
        raise ValueError(f"q heads have {dim} elements, the cache's {key_dim}")
    _expect_rows(block_tables, "block_tables", torch.int32, 2, device)
    requests, max_blocks = block_tables.shape
    _expect_all(device, ((query_start, "query_start", torch.int32, (requests + 1,)),
                         (kv_lens, "kv_lens", torch.int32, (requests,))))
    if scale is None:
        scale = ctypes.c_float(dim ** -0.5).value
    if out is None:
        out = q.new_empty((tokens, query_heads * dim))
    else:
        _expect_all(device, ((out, "out", BF16, (tokens, query_heads * dim)),))
    _ready(q)
    lib = _lib.library()
    max_query_len, max_kv_len = int(max_query_len), int(max_kv_len)
    need = lib.aoto_hip_paged_attention_workspace(tokens, requests, max_blocks, page, query_heads, kv_heads, dim,
                                                  max_query_len, max_kv_len)
    if workspace is not None:
        _on_device(workspace)
        if workspace.get_device() != device:
            raise ValueError(f"the workspace is on {workspace.device}, the call's other tensors on cuda:{device}")
        if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
            workspace = None
    if need and workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=q.device)
    _lib.check(
        lib.aoto_hip_paged_attention(
            _ptr(q), q.stride(0), q.stride(1), _ptr(keys), _ptr(values), page_stride, head_stride,
            slot_stride, pages, page, _ptr(block_tables), block_tables.stride(0), max_blocks, _ptr(query_start),
            _ptr(kv_lens), tokens, requests, query_heads, kv_heads, dim, int(bool(causal)), float(scale),
            max_query_len, max_kv_len, _ptr(workspace if need else None), _ptr(out), _stream(device),
        )
    )
    return out


def verify_draft(
    logits: torch.Tensor,
    draft_tokens: torch.Tensor,
    query_start: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    draft_logits: torch.Tensor | None = None,
    temperature: torch.Tensor | None = None,
    tokens: torch.Tensor | None = None,
    accepted: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Drafted tokens against the target's logits: ``(tokens [R, K + 1] int64, accepted [R] int32)``.

    Rows ``query_start[r] .. query_start[r + 1]`` of ``logits [T, V]`` (bf16 or f32) judge the first drafts of
    ``draft_tokens[r]`` (int64 ``[R, K]``, ``K <= 62``) one row each; the last row follows them all (no drafts: plain
    sampling). With ``p`` the softmax of a row at ``temperature[r]`` (f32 ``[R]``), ``q`` that of its draft's
    ``draft_logits[r, i]`` (``[R, K, V]`` of the logits' type; None: the draft is certain) and ``u = uniforms[r]``
    (f32 ``[R, K + 1]`` in [0, 1)), draft ``x`` stands while ``u[i] * q[x] < p[x]``. The token after those that stand
    is drawn with ``u[K]`` from ``max(p - q, 0)`` of the first that fell, or from the last row's ``p``: the first one
    at which the running sum of weights is above ``u[K]`` times their total. At a temperature of 0 (and everywhere
    with ``temperature=None``) a draft stands where it is the row's first maximum, which is also the token that
    follows. ``tokens`` holds the drafts that stand, the token that follows them and -1 behind it; ``accepted`` counts
    the former. A request without rows gets -1 throughout. Weights and sums are held in 64 bits (the exponentials right
    to 3e-15 of themselves).
    """

    dtype = logits.dtype if isinstance(logits, torch.Tensor) else BF16
    if dtype not in (BF16, torch.float32):
        raise TypeError(f"logits must be bf16 or f32, got {dtype}")
    _expect_rows(logits, "logits", dtype, 2, logits.get_device() if isinstance(logits, torch.Tensor) else 0)
    device = _on_current("logits", logits)
    rows, vocab = logits.shape
    _expect_all(device, ((draft_tokens, "draft_tokens", torch.int64, None),))
    if draft_tokens.dim() != 2:
        raise ValueError(f"draft_tokens must be [R, K], got {tuple(draft_tokens.shape)}")
    requests, drafts = draft_tokens.shape
    _expect_all(device, ((query_start, "query_start", torch.int32, (requests + 1,)),
                         (uniforms, "uniforms", torch.float32, (requests, drafts + 1))))
    if temperature is not None:
        _expect_all(device, ((temperature, "temperature", torch.float32, (requests,)),))
    if draft_logits is not None:
        _expect_rows(draft_logits, "draft_logits", dtype, 3, device)
        if tuple(draft_logits.shape) != (requests, drafts, vocab):
            raise ValueError(f"draft_logits must be {(requests, drafts, vocab)}, got {tuple(draft_logits.shape)}")
    if tokens is None:
        tokens = draft_tokens.new_empty((requests, drafts + 1))
    else:
        _expect_all(device, ((tokens, "tokens", torch.int64, (requests, drafts + 1)),))
    if accepted is None:
        accepted = query_start.new_empty((requests,))
    else:
        _expect_all(device, ((accepted, "accepted", torch.int32, (requests,)),))
    _ready(logits)
    lib = _lib.library()
    need = lib.aoto_hip_verify_draft_workspace(requests, drafts, vocab)
    if workspace is not None:
        _on_device(workspace)
        if workspace.get_device() != device:
            raise ValueError(f"the workspace is on {workspace.device}, the call's other tensors on cuda:{device}")
        if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
            workspace = None
    if workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=logits.device)
    _lib.check(
        lib.aoto_hip_verify_draft(
            _ptr(logits), int(dtype is torch.float32), logits.stride(0), rows, vocab, _ptr(draft_tokens),
            _ptr(draft_logits), 0 if draft_logits is None else draft_logits.stride(0),
            0 if draft_logits is None else draft_logits.stride(1), _ptr(query_start), _ptr(uniforms),
            _ptr(temperature), requests, drafts, _ptr(workspace), _ptr(tokens), _ptr(accepted), _stream(device),
        )
    )
    return tokens, accepted


# ------------------------------------------------------------------------------------------------------------------
# The functions from here on make their call through ``_calls`` (csrc/calls.cpp) where that is built: the checks, the
# outputs' allocation and the C ABI's call in one step (an attention's call takes 5.7 us with its launch, 11.4 below).
# It gives None where an argument is not as it should be or the call was refused; the checks below then say why, or make
# a call that it does not (outputs given as a tuple, numbers of other types).


class _Unbound:
    """``_calls`` before it is bound, and where it is not built: makes no call."""

    def __getattr__(self, name: str):
        return lambda *args: None


class _Refused(_Unbound):
    """The same in place of a build that is not to be bound."""


_calls = _Unbound()

#: The entry points ``_calls`` is given, in its order.
_CALLED = ("code_object_loaded", "paged_rope_append_mx4", "paged_unpack_mx4", "paged_attention_mx4",
           "paged_attention_mx4_workspace", "paged_fork", "paged_release", "paged_compact", "paged_copy",
           "adjust_logits")


def _bind_calls() -> None:
    """Bind ``_calls``, once, on the way of a first call that was made without it."""

    global _calls
    if type(_calls) is not _Unbound or _raw_stream is None:
        return
    try:
        from . import _calls as module
    except ImportError:
        return
    from .csrc.build import calls_built_for

    if getattr(module, "built_for", None) != calls_built_for():  # the layout of its tensors may be another
        warnings.warn("_calls.so is of another build of torch or Python, the calls are made without it: build it with "
                      "`python -m aotolith_amd.csrc.build`")
        _calls = _Refused()
        return
    lib = _lib.library()
    entries = (ctypes.cast(getattr(lib, "aoto_hip_" + name), ctypes.c_void_p).value for name in _CALLED)
    module.bind(*entries, _raw_stream, PagedMx4, _lib.check)
    _calls = module


# ------------------------------------------------------------------------------------------------------------------
# The paged cache in 4 bits. A row of D dims is D / 2 bytes of codes and D / 32 scale bytes: a code is a sign and one of
# 0, 0.5, 1, 1.5, 2, 3, 4, 6 (dim 2i in the low half of byte i), its group of 32 dims shares the scale 2^(byte - 127),
# and a byte above 252 makes the group NaN. 68 bytes for 128 dims, 256 in bf16.


class PagedMx4(NamedTuple):
    """A layer's cache in 4 bits: uint8 codes ``[pages, Hkv, page, D / 2]`` and scale bytes ``[pages, Hkv, page,
    D / 32]`` (views with contiguous rows will do; the codes' other strides and bases are multiples of 16 bytes)."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor


def paged_mx4_cache(pages: int, kv_heads: int, page_size: int, head_dim: int, *, device=None) -> PagedMx4:
    """A layer's cache in 4 bits, all zeros."""

    pages, kv_heads, page_size, head_dim = int(pages), int(kv_heads), int(page_size), int(head_dim)
    if min(pages, kv_heads, page_size, head_dim) <= 0 or head_dim % 64:
        raise ValueError("a 4-bit cache has heads of multiples of 64 dims, got "
                         f"{pages} pages of {kv_heads} x {page_size} rows of {head_dim}")
    device = torch.device("cuda") if device is None else device
    codes, scales = (torch.zeros((2, pages, kv_heads, page_size, head_dim // n), dtype=torch.uint8, device=device)
                     for n in (2, 32))
    return PagedMx4(*codes.unbind(), *scales.unbind())


def _expect_mx4(cache: PagedMx4, device: int) -> tuple[tuple, bytes]:
    """``(pages, Hkv, page, D)`` of a cache, and its descriptor for the C ABI."""

    if not isinstance(cache, PagedMx4):
        raise TypeError(f"cache must be a PagedMx4, got {type(cache).__name__}")
    keys, values, key_scales, value_scales = cache
    u8 = torch.uint8
    try:  # one pass over the attributes, the reasons only for a cache that fails
        shape, strides, small, scale_strides = keys.shape, keys.stride(), key_scales.shape, key_scales.stride()
        pages, kv_heads, page, half = shape
        good = (keys.dtype is u8 and values.dtype is u8 and key_scales.dtype is u8 and value_scales.dtype is u8
                and keys.get_device() == device and values.get_device() == device
                and key_scales.get_device() == device and value_scales.get_device() == device
                and values.shape == shape and values.stride() == strides and strides[3] == 1
                and small == (pages, kv_heads, page, half // 16) and half % 32 == 0
                and value_scales.shape == small and value_scales.stride() == scale_strides and scale_strides[3] == 1)
    except (AttributeError, ValueError):
        good = False
    if not good:
        for name, tensor in zip(cache._fields, cache):
            _expect_rows(tensor, name, u8, 4, device)
        shape, strides, scale_strides = keys.shape, keys.stride(), key_scales.stride()
        if shape != values.shape or strides != values.stride():
            raise ValueError("keys and values must have one shape and the same strides")
        pages, kv_heads, page, half = shape
        if half % 32:
            raise ValueError(f"heads of a 4-bit cache have a multiple of 64 dims, got {2 * half}")
        want = (pages, kv_heads, page, half // 16)
        if tuple(key_scales.shape) != want or tuple(value_scales.shape) != want:
            raise ValueError(f"key_scales and value_scales must be {want}, got {tuple(key_scales.shape)} and "
                             f"{tuple(value_scales.shape)}")
        if scale_strides != value_scales.stride():
            raise ValueError("key_scales and value_scales must have the same strides")
    return (pages, kv_heads, page, 2 * half), _lib.MX4_CACHE.pack(
        keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), *strides[:3],
        *scale_strides[:3], pages)


def paged_rope_append_mx4(
    qkv: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    cache: PagedMx4,
    *,
    query_heads: int,
    q_out: torch.Tensor | None = None,
    error: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_rope_append` into a 4-bit cache: returns ``q [T, Hq, D]``.

    Keys go from f32 to their codes without a rounding to bf16 between. A group's scale is the least power of two of
    which its largest magnitude is at most 7 (bytes 1 to 252), a code the nearest value, ties to the even code,
    magnitudes above 6 to 6; a group that holds an infinity or a NaN stands for NaN.
    """

    made = _calls.paged_rope_append_mx4(qkv, positions, slots, cos_table, sin_table, cache, query_heads, q_out, error)
    if made is not None:
        return made

    _expect_rows(qkv, "qkv", BF16, 2, qkv.get_device() if isinstance(qkv, torch.Tensor) else 0)
    device = _on_current("qkv", qkv)
    (_, kv_heads, page, dim), arg = _expect_mx4(cache, device)
    tokens, width = qkv.shape
    query_heads = int(query_heads)
    if query_heads <= 0 or width != (query_heads + 2 * kv_heads) * dim:
        raise ValueError(f"qkv rows of {width} do not hold {query_heads} + 2 x {kv_heads} heads of {dim}")
    _expect_all(device, ((positions, "positions", torch.int64, (tokens,)), (slots, "slots", torch.int64, (tokens,)),
                         (cos_table, "cos_table", BF16, None)))
    if cos_table.dim() != 2 or cos_table.shape[1] != dim:
        raise ValueError(f"cos_table must be [P, {dim}], got {tuple(cos_table.shape)}")
    _expect_all(device, ((sin_table, "sin_table", BF16, cos_table.shape),))
    if error is not None:
        _expect_all(device, ((error, "error", torch.int32, (1,)),))
    if q_out is None:
        q_out = qkv.new_empty((tokens, query_heads, dim))
    else:
        _expect_all(device, ((q_out, "q_out", BF16, (tokens, query_heads, dim)),))
    _ready(qkv)
    _bind_calls()
    _lib.check(
        _lib.library().aoto_hip_paged_rope_append_mx4(
            _ptr(qkv), qkv.stride(0), _ptr(positions), _ptr(slots), _ptr(cos_table), _ptr(sin_table),
            cos_table.shape[0], arg, page, tokens, query_heads, kv_heads, dim, _ptr(q_out), _ptr(error),
            _stream(device),
        )
    )
    return q_out


def paged_unpack_mx4(cache: PagedMx4, *, out: tuple[torch.Tensor, torch.Tensor] | None = None
                     ) -> tuple[torch.Tensor, torch.Tensor]:
    """What a 4-bit cache stands for: ``(keys, values)`` bf16 ``[pages, Hkv, page, D]`` (exact: bf16 holds every value
    that an append writes)."""

    if out is None:
        made = _calls.paged_unpack_mx4(cache)
        if made is not None:
            return made

    if not isinstance(cache, PagedMx4):
        raise TypeError(f"cache must be a PagedMx4, got {type(cache).__name__}")
    _expect_rows(cache.keys, "keys", torch.uint8, 4, cache.keys.get_device()
                 if isinstance(cache.keys, torch.Tensor) else 0)
    device = _on_current("keys", cache.keys)
    shape, arg = _expect_mx4(cache, device)
    if out is None:
        out = torch.empty((2, *shape), dtype=BF16, device=cache.keys.device).unbind()
    else:
        keys_out, values_out = out
        _expect_all(device, ((keys_out, "out[0]", BF16, shape), (values_out, "out[1]", BF16, shape)))
    _ready(cache.keys)
    _bind_calls()
    _lib.check(_lib.library().aoto_hip_paged_unpack_mx4(arg, shape[2], shape[1], shape[3], _ptr(out[0]),
                                                        _ptr(out[1]), _stream(device)))
    return out


def paged_attention_mx4_workspace(tokens: int, requests: int, max_blocks: int, page_size: int, query_heads: int,
                                  kv_heads: int, head_dim: int, *, max_query_len: int = 0, max_kv_len: int = 0,
                                  device=None) -> torch.Tensor:
    """A workspace for :func:`paged_attention_mx4` with these shapes and bounds, as
    :func:`paged_attention_workspace`'s."""

    size = _lib.library().aoto_hip_paged_attention_mx4_workspace(
        int(tokens), int(requests), int(max_blocks), int(page_size), int(query_heads), int(kv_heads), int(head_dim),
        int(max_query_len), int(max_kv_len))
    return torch.empty((max(size, 16),), dtype=torch.uint8, device=device)


def paged_attention_mx4(
    q: torch.Tensor,
    cache: PagedMx4,
    block_tables: torch.Tensor,
    query_start: torch.Tensor,
    kv_lens: torch.Tensor,
    *,
    causal: bool = True,
    scale: float | None = None,
    max_query_len: int = 0,
    max_kv_len: int = 0,
    workspace: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_attention` over a 4-bit cache: the requests' new tokens ``q [T, Hq, D]`` (D 64 or 128) over the
    values that the codes of their pages stand for -> ``[T, Hq * D]``.

    Everything else is :func:`paged_attention`'s, what a row sees among it (the workspace:
    :func:`paged_attention_mx4_workspace`). A NaN group of a key that a row sees, a NaN or an infinity in its q make
    the row NaN; a NaN group of a value makes those 32 dims NaN, however small its weight. Requests of more than 32 rows
    a kv head multiply K as it is in the cache by q as two 8-bit numbers (exactly q to 2^-22 of the largest of each 32
    dims), in sums that keep 13 bits below the largest of each eight products. Scores are of magnitudes below 2^29: past
    it the exponentials lose their reference, which is held in f32.
    """

    made = _calls.paged_attention_mx4(q, cache, block_tables, query_start, kv_lens, causal, scale, max_query_len,
                                      max_kv_len, workspace, out)
    if made is not None:
        return made

    _expect_rows(q, "q", BF16, 3, q.get_device() if isinstance(q, torch.Tensor) else 0)
    device = _on_current("q", q)
    tokens, query_heads, dim = q.shape
    (_, kv_heads, page, key_dim), arg = _expect_mx4(cache, device)
    if key_dim != dim:
        raise ValueError(f"q heads have {dim} elements, the cache's {key_dim}")
    _expect_rows(block_tables, "block_tables", torch.int32, 2, device)
    requests, max_blocks = block_tables.shape
    _expect_all(device, ((query_start, "query_start", torch.int32, (requests + 1,)),
                         (kv_lens, "kv_lens", torch.int32, (requests,))))
    if scale is None:
        scale = ctypes.c_float(dim ** -0.5).value
    if out is None:
        out = q.new_empty((tokens, query_heads * dim))
    else:
        _expect_all(device, ((out, "out", BF16, (tokens, query_heads * dim)),))
    _ready(q)
    _bind_calls()
    lib = _lib.library()
    max_query_len, max_kv_len = int(max_query_len), int(max_kv_len)
    if not (0 <= max_query_len < 2 ** 31 and 0 <= max_kv_len < 2 ** 31):
        raise ValueError(f"max_query_len and max_kv_len are of 31 bits, got {max_query_len} and {max_kv_len}")
    need = lib.aoto_hip_paged_attention_mx4_workspace(tokens, requests, max_blocks, page, query_heads, kv_heads, dim,
                                                      max_query_len, max_kv_len)
    if workspace is not None:
        _on_device(workspace)
        if workspace.get_device() != device:
            raise ValueError(f"the workspace is on {workspace.device}, the call's other tensors on cuda:{device}")
        if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
            workspace = None
    if need and workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=q.device)
    _lib.check(
        lib.aoto_hip_paged_attention_mx4(
            _ptr(q), q.stride(0), q.stride(1), arg, page, _ptr(block_tables), block_tables.stride(0),
            max_blocks, _ptr(query_start), _ptr(kv_lens), tokens, requests, query_heads, kv_heads, dim,
            int(bool(causal)), float(scale), max_query_len, max_kv_len, _ptr(workspace if need else None), _ptr(out),
            _stream(device),
        )
    )
    return out


# ------------------------------------------------------------------------------------------------------------------
# The pages of a cache beyond a step's own. ``shares`` (int32 ``[pages]``) counts a page's holders beyond the first: the
# block table rows that name it within their page counts. :func:`paged_tables` takes pages that nobody shares.

#: More bits of the ``error`` tensor, raised by the functions below (``AOTO_PAGED_*`` in ``include/aoto_hip.h``).
PAGED_ROW_HELD, PAGED_BAD_ROW, PAGED_BAD_SHARE, PAGED_LIST_FULL, PAGED_ROW_SHARED = 32, 64, 128, 256, 512


class PagedFork(NamedTuple):
    """What :func:`paged_fork` says of the requests, and the pages to copy."""

    context_lens: torch.Tensor  # int32 [R]
    page_counts: torch.Tensor   # int32 [R]
    free_start: torch.Tensor    # int32 [1]
    source: torch.Tensor        # int32 [R]: the page to copy for each row, -1 without
    target: torch.Tensor        # int32 [R]: where to


class PagedMoves(NamedTuple):
    """What :func:`paged_compact` moved: page ``source[i]`` to ``target[i]``, ``i < count``; -1 behind them."""

    source: torch.Tensor  # int32 [pages]
    target: torch.Tensor  # int32 [pages]
    count: torch.Tensor   # int32 [1]


def _page_size(page_size: int) -> int:
    """For the C ABI's 32 bits, which ctypes cuts an integer to without a word."""

    page_size = int(page_size)
    if not -(2 ** 31) <= page_size < 2 ** 31:
        raise ValueError(f"page_size is a number of 32 bits, got {page_size}")
    return page_size


def _expect_pool(block_tables, page_counts, shares, free_pages, free_start, error) -> tuple[int, int]:
    """The pool's tensors, as every function on pages takes them: ``(device, requests)``."""

    _expect(shares, "shares", torch.int32)
    device = _on_current("shares", shares)
    if shares.dim() != 1 or not shares.numel():
        raise ValueError(f"shares must be [pages], got {tuple(shares.shape)}")
    _expect_rows(block_tables, "block_tables", torch.int32, 2, device)
    requests = block_tables.shape[0]
    _expect_all(device, (
        (page_counts, "page_counts", torch.int32, (requests,)), (free_pages, "free_pages", torch.int32, None),
        (free_start, "free_start", torch.int32, (1,)),
    ))
    if error is not None:
        _expect_all(device, ((error, "error", torch.int32, (1,)),))
    return device, requests


def paged_fork(
    parents: torch.Tensor,
    context_lens: torch.Tensor,
    block_tables: torch.Tensor,
    page_counts: torch.Tensor,
    shares: torch.Tensor,
    free_pages: torch.Tensor,
    free_start: torch.Tensor,
    *,
    page_size: int,
    step: PagedFork | None = None,
    error: torch.Tensor | None = None,
) -> PagedFork:
    """Requests that go on from another: samples of one prompt, beams.

    Row ``r`` with ``parents[r] >= 0`` (int32 ``[R]``) must hold no pages; it gets the cached tokens of row
    ``parents[r]`` as that was before the call. Full pages are shared: entered in its row of ``block_tables``, one more
    in ``shares``. A page in progress becomes the next one of ``free_pages[free_start:]``, rows in order, and its
    content is to be copied: ``source``, ``target`` for :func:`paged_copy` on every layer's cache. Other rows stay, but
    for the page that one of ``context_lens[r]`` tokens has in progress: where others hold it too (:func:`paged_release`
    cut the row there), the row gets a page of its own in its place, with the copy in ``source`` and ``target``, before
    tokens that are appended would become the others'. (The last holder that ends there keeps the page.)
    ``block_tables`` and ``shares`` are changed in place; lengths, counts and the list's start are in the result, whose
    tensors ``step`` may give: these three also as the ones passed in, else in memory of their own. ``error`` (int32
    ``[1]``) collects ``PAGED_ROW_HELD`` (the row holds pages: left as it is), ``PAGED_BAD_ROW`` (no such parent: the
    same), ``PAGED_NO_PAGES`` (the free list ran out: the row ends with its last full page) and ``PAGED_ROW_SHARED``
    (nor was there a page for a row that ends inside another's: it is as it was and must not be appended to).
    """

    if step is None:
        made = _calls.paged_fork(parents, context_lens, block_tables, page_counts, shares, free_pages, free_start,
                                 page_size, error)
        if made is not None:
            return PagedFork(*made)

    device, requests = _expect_pool(block_tables, page_counts, shares, free_pages, free_start, error)
    _expect_all(device, ((parents, "parents", torch.int32, (requests,)),
                         (context_lens, "context_lens", torch.int32, (requests,))))
    shapes = ((requests,), (requests,), (1,), (requests,), (requests,))
    if step is None:
        all_of = shares.new_empty((6 * requests + 1,))
        lens, counts, source, target, plan, first = all_of.split_with_sizes(
            (requests, requests, requests, requests, 2 * requests, 1))
        step = PagedFork(lens, counts, first, source, target)
    else:
        _expect_all(device, ((x, f"step.{name}", torch.int32, shape)
                             for x, name, shape in zip(step, PagedFork._fields, shapes)))
        plan = shares.new_empty((2 * requests,))
    _ready(shares)
    _bind_calls()
    _lib.check(
        _lib.library().aoto_hip_paged_fork(
            _ptr(parents), _ptr(context_lens), _ptr(block_tables), block_tables.stride(0), _ptr(page_counts),
            _ptr(shares), _ptr(free_pages), _ptr(free_start), requests, block_tables.shape[1], free_pages.numel(),
            shares.numel(), _page_size(page_size), _ptr(step.context_lens), _ptr(step.page_counts),
            _ptr(step.free_start), _ptr(step.source), _ptr(step.target), _ptr(plan), _ptr(error), _stream(device),
        )
    )
    return step


def paged_release(
    keep_lens: torch.Tensor,
    block_tables: torch.Tensor,
    page_counts: torch.Tensor,
    shares: torch.Tensor,
    free_pages: torch.Tensor,
    free_start: torch.Tensor,
    *,
    page_size: int,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
    error: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages given back, of requests that ended or whose drafted tokens did not stand: ``(page_counts, free_start)``.

    Row ``r`` keeps the pages of its first ``keep_lens[r]`` tokens (int32 ``[R]``; 0: none, negative: all that it has).
    The others lose a holder each, and those left without one go to the places of ``free_pages`` before ``free_start``,
    downwards from it in ascending order of their numbers. ``shares`` and ``free_pages`` are changed in place, entries
    of ``block_tables`` past the new counts stay what they were; ``out`` gives the tensors of the result, which may be
    the ones passed in. ``error`` (int32 ``[1]``) collects ``PAGED_BAD_SHARE`` (a page given back more often than held,
    in this call or by one before: what ``free_pages[free_start:]`` holds already is not entered again) and
    ``PAGED_LIST_FULL`` (no place before the list's first: the page is lost).

    A row that went on from another may be cut inside a page that it still shares. The next token's slot is in that
    page, over the others' tokens: :func:`paged_fork` (with ``parents`` of -1 where no row goes on) and its copy come
    before the step's :func:`paged_tables`, and give the row a page of its own. (With ``shares``, that call leaves such
    tokens out and says so.)
    """

    if out is None:
        made = _calls.paged_release(keep_lens, block_tables, page_counts, shares, free_pages, free_start, page_size,
                                    error)
        if made is not None:
            return made

    device, requests = _expect_pool(block_tables, page_counts, shares, free_pages, free_start, error)
    _expect_all(device, ((keep_lens, "keep_lens", torch.int32, (requests,)),))
    room = shares.numel() // 1024 + 2
    if out is None:
        counts_out, start_out, scratch = shares.new_empty((requests + 1 + room,)).split_with_sizes((requests, 1, room))
    else:
        counts_out, start_out = out
        scratch = shares.new_empty((room,))
        _expect_all(device, ((counts_out, "out[0]", torch.int32, (requests,)),
                             (start_out, "out[1]", torch.int32, (1,))))
    _ready(shares)
    _bind_calls()
    _lib.check(
        _lib.library().aoto_hip_paged_release(
            _ptr(keep_lens), _ptr(block_tables), block_tables.stride(0), _ptr(page_counts), _ptr(shares),
            _ptr(free_pages), _ptr(free_start), requests, block_tables.shape[1], free_pages.numel(), shares.numel(),
            _page_size(page_size), _ptr(counts_out), _ptr(start_out), _ptr(scratch), _ptr(error), _stream(device),
        )
    )
    return counts_out, start_out


def paged_compact(
    block_tables: torch.Tensor,
    page_counts: torch.Tensor,
    shares: torch.Tensor,
    free_pages: torch.Tensor,
    free_start: torch.Tensor,
    *,
    moves: PagedMoves | None = None,
    error: torch.Tensor | None = None,
) -> PagedMoves:
    """A pool's pages moved together, so that what is behind them can be given up.

    With ``m`` pages held by the rows of ``block_tables`` and the pages held or in ``free_pages[free_start:]`` in
    ascending order, held pages past the first ``m`` of them go, in order, to free ones among the first ``m``. The
    tables and ``shares`` are changed to the new numbers in place; the free list keeps its place and holds the rest,
    ascending (so the pool's highest numbers are free ones). Pages neither held nor free stay what they are. The
    contents are :func:`paged_copy`'s, on every layer's cache, with the result's ``source``, ``target`` and ``count``
    (tensors that ``moves`` may give, in memory of their own).
    ``error`` (int32 ``[1]``) collects ``PAGED_BAD_SHARE``: a page both held and free, or a list that names a page twice
    or none.
    """

    if moves is None:
        made = _calls.paged_compact(block_tables, page_counts, shares, free_pages, free_start, error)
        if made is not None:
            return PagedMoves(*made)

    device, requests = _expect_pool(block_tables, page_counts, shares, free_pages, free_start, error)
    pages = shares.numel()
    if moves is None:
        source, target, state, count = shares.new_empty((3 * pages + 1,)).split_with_sizes((pages, pages, pages, 1))
        moves = PagedMoves(source, target, count)
    else:
        _expect_all(device, ((x, f"moves.{name}", torch.int32, shape)
                             for x, name, shape in zip(moves, PagedMoves._fields, ((pages,), (pages,), (1,)))))
        state = shares.new_empty((pages,))
    _ready(shares)
    _bind_calls()
    _lib.check(
        _lib.library().aoto_hip_paged_compact(
            _ptr(block_tables), block_tables.stride(0), _ptr(page_counts), _ptr(shares), _ptr(free_pages),
            _ptr(free_start), requests, block_tables.shape[1], free_pages.numel(), pages, _ptr(moves.source),
            _ptr(moves.target), _ptr(moves.count), _ptr(state), _ptr(error), _stream(device),
        )
    )
    return moves


def _page_tensor(tensor: torch.Tensor, index: int, dim: int, pages: int | None, device: int) -> bytes:
    name = f"caches[{index}]"
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(tensor).__name__}")
    if tensor.device.type != "cuda":
        raise ValueError(f"{name} must be on the GPU, got {tensor.device}")
    if tensor.get_device() != device:
        raise ValueError(f"{name} is on {tensor.device}, the call's other tensors on cuda:{device}")
    shape, strides, size = tensor.shape, tensor.stride(), tensor.element_size()
    if not 0 <= dim < len(shape) or not tensor.numel():
        raise ValueError(f"{name} {tuple(shape)} has no pages in dim {dim}")
    if pages is not None and shape[dim] != pages:
        raise ValueError(f"{name} has {shape[dim]} pages, the first tensor {pages}")
    # a page: its dims in some order one dense block
    dense = 1
    for stride, length in sorted((s, n) for s, n in zip(strides[dim + 1:], shape[dim + 1:]) if n > 1):
        if stride != dense:
            raise ValueError(f"{name}'s pages must be dense in memory, got strides {strides}")
        dense *= length
    planes, plane_stride = 1, 0
    for stride, length in zip(strides[:dim][::-1], shape[:dim][::-1]):
        if length == 1:
            continue
        if planes > 1 and stride != planes * plane_stride:
            raise ValueError(f"{name}'s dims before its pages must be evenly spaced, got strides {strides}")
        plane_stride = plane_stride if planes > 1 else stride
        planes *= length
    page_stride = strides[dim] if shape[dim] > 1 else dense
    # of two strides the smaller one is past a page, the other past all that it spans
    low, high = sorted(((page_stride, shape[dim]), (plane_stride if planes > 1 else page_stride * shape[dim], planes)))
    if low[0] < dense or high[0] < low[0] * (low[1] - 1) + dense:
        raise ValueError(f"{name}'s pages overlap, got strides {strides}")
    return _lib.PAGE_TENSOR.pack(tensor.data_ptr(), planes, plane_stride * size, page_stride * size, dense * size)


def paged_copy(
    caches: torch.Tensor | list[torch.Tensor] | tuple[torch.Tensor, ...],
    source: torch.Tensor,
    target: torch.Tensor,
    *,
    count: torch.Tensor | None = None,
    dim: int = 0,
    error: torch.Tensor | None = None,
) -> None:
    """Pages' contents from ``source[i]`` to ``target[i]`` (int32 ``[N]``) in every tensor of ``caches``, in place.

    The pages are in dim ``dim`` of each tensor, of any type: ``[pages, Hkv, page, D]`` for one layer's keys, with
    ``dim=2`` ``[layers, 2, pages, ...]`` for all layers at once. What follows that dim is dense in memory (in any
    order), what precedes it evenly spaced. ``count`` (int32 ``[1]``, on the GPU) takes only the first pairs. Pairs with
    a -1 are left out, and others that name no page too, which raises ``PAGED_BAD_SLOT`` in ``error`` (int32 ``[1]``).
    No target may be the source or the target of another pair, as none of :func:`paged_fork` and :func:`paged_compact`
    is.
    """

    if _calls.paged_copy(caches, source, target, count, dim, error) is not None:
        return

    _expect(source, "source", torch.int32)
    device = _on_current("source", source)
    if source.dim() != 1:
        raise ValueError(f"source must be [N], got {tuple(source.shape)}")
    _expect_all(device, ((target, "target", torch.int32, source.shape),))
    for x, name in ((count, "count"), (error, "error")):
        if x is not None:
            _expect_all(device, ((x, name, torch.int32, (1,)),))
    if isinstance(caches, torch.Tensor):
        caches = (caches,)
    if not caches:
        raise ValueError("no caches")
    dim = int(dim)
    args, pages = [], None
    for i, tensor in enumerate(caches):
        args.append(_page_tensor(tensor, i, dim, pages, device))
        pages = tensor.shape[dim]
    if not source.numel():
        return
    _ready(source)
    _bind_calls()
    _lib.check(
        _lib.library().aoto_hip_paged_copy(
            b"".join(args), len(args), pages, _ptr(source), _ptr(target), source.numel(), _ptr(count), _ptr(error),
            _stream(device),
        )
    )


def adjust_logits(
    logits: torch.Tensor,
    query_start: torch.Tensor | None = None,
    *,
    history: torch.Tensor | None = None,
    history_lens: torch.Tensor | None = None,
    prompt_lens: torch.Tensor | None = None,
    draft_tokens: torch.Tensor | None = None,
    repetition: torch.Tensor | None = None,
    presence: torch.Tensor | None = None,
    frequency: torch.Tensor | None = None,
    bias_tokens: torch.Tensor | None = None,
    bias_values: torch.Tensor | None = None,
    allowed: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Penalties, biases and masks on ``logits [T, V]`` (bf16 or f32), before :func:`verify_draft` judges or draws.

    Request ``r`` has the rows ``query_start[r] .. query_start[r + 1]`` (int32 ``[R + 1]``; None: one row each), row
    ``i`` of them behind its first ``i`` drafts (``draft_tokens`` int64 ``[R, K]``). Its text is ``history[r]`` (int64
    ``[R, L]``) up to ``history_lens[r]`` (int32 ``[R]``; None: L), from ``prompt_lens[r]`` on (None: 0) its own answer,
    and those drafts, which belong to the answer. In this order, in f32, with one rounding:

    * a logit ``z`` of a token in the text becomes ``z / repetition[r]`` if positive, else ``z * repetition[r]``,
    * that of a token ``c > 0`` times in the answer loses ``frequency[r] * c + presence[r]``,
    * ``bias_values[r, j]`` is added to that of ``bias_tokens[r, j]`` (f32 and int64 ``[R, B]``, the last entry of a
      token counts, tokens outside the vocabulary, -1 say, are none),
    * one whose bit ``v % 32`` of ``allowed[t, v // 32]`` (int32 ``[T, ceil(V / 32)]``) is 0 becomes -inf.

    ``repetition``, ``presence``, ``frequency`` are f32 ``[R]``; what is None is left out. ``out`` may be ``logits``;
    its rows of no request are left as they are (in a new tensor: not set).
    """

    made = _calls.adjust_logits(logits, query_start, history, history_lens, prompt_lens, draft_tokens, repetition,
                                presence, frequency, bias_tokens, bias_values, allowed, out)
    if made is not None:
        return made

    dtype = logits.dtype if isinstance(logits, torch.Tensor) else BF16
    if dtype not in (BF16, torch.float32):
        raise TypeError(f"logits must be bf16 or f32, got {dtype}")
    _expect_rows(logits, "logits", dtype, 2, logits.get_device() if isinstance(logits, torch.Tensor) else 0)
    device = _on_current("logits", logits)
    rows, vocab = logits.shape
    requests = rows
    if query_start is not None:
        _expect_all(device, ((query_start, "query_start", torch.int32, None),))
        requests = query_start.numel() - 1
        if query_start.dim() != 1 or requests < 1:
            raise ValueError(f"query_start must be [R + 1], got {tuple(query_start.shape)}")
    def lists(tensor, name, kind, rows_, columns=None):
        """A ``[rows_, columns]`` operand's address, row stride and columns."""

        _expect_rows(tensor, name, kind, 2, device)
        shape = tensor.shape
        if shape[0] != rows_ or columns is not None and shape[1] != columns:
            raise ValueError(f"{name} must be {(rows_, shape[1] if columns is None else columns)}, got {tuple(shape)}")
        return tensor.data_ptr(), tensor.stride(0), shape[1]

    def each(tensor, name, kind):
        """A ``[R]`` operand's address."""

        if tensor is None:
            return 0
        _expect_all(device, ((tensor, name, kind, (requests,)),))
        return tensor.data_ptr()

    none = (0, 0, 0)
    if history is None and (history_lens is not None or prompt_lens is not None):
        raise ValueError("history_lens and prompt_lens need a history")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values come together")
    text = none if history is None else lists(history, "history", torch.int64, requests)
    drafts = none if draft_tokens is None else lists(draft_tokens, "draft_tokens", torch.int64, requests)
    biases = none if bias_tokens is None else lists(bias_tokens, "bias_tokens", torch.int64, requests)
    values = none if bias_values is None else lists(bias_values, "bias_values", torch.float32, requests, biases[2])
    masks = none if allowed is None else lists(allowed, "allowed", torch.int32, rows, (vocab + 31) // 32)
    arg = _lib.ADJUSTMENTS.pack(
        0 if query_start is None else query_start.data_ptr(), text[0], each(history_lens, "history_lens", torch.int32),
        each(prompt_lens, "prompt_lens", torch.int32), drafts[0], each(repetition, "repetition", torch.float32),
        each(presence, "presence", torch.float32), each(frequency, "frequency", torch.float32), biases[0], values[0],
        masks[0], text[1], drafts[1], biases[1], values[1], masks[1], text[2], drafts[2], biases[2])
    if out is None:
        out = logits.new_empty((rows, vocab))
    else:
        _expect_rows(out, "out", dtype, 2, device)
        if out.shape != logits.shape:
            raise ValueError(f"out must be {(rows, vocab)}, got {tuple(out.shape)}")
        if rows > 1 and out.stride(0) < vocab:
            raise ValueError(f"out's rows overlap, got strides {out.stride()}")
        if (out.untyped_storage().data_ptr() == logits.untyped_storage().data_ptr()
                and (out.data_ptr() != logits.data_ptr() or out.stride() != logits.stride())):
            raise ValueError("out must be logits itself or in memory of its own")
    _ready(logits)
    _bind_calls()
    _lib.check(
        _lib.library().aoto_hip_adjust_logits(
            _ptr(logits), int(dtype is torch.float32), logits.stride(0), rows, vocab, requests, arg,
            _ptr(out), out.stride(0), _stream(device),
        )
    )
    return out
