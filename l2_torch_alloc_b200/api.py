"""Host-side mirror of the reference's Python interface (example_wrapper.py:1-187,
test.py:41-157), rewritten around a small class so several users can share one
loaded library.  Argument names, meanings and assertion behaviour follow the
reference; the known slip there (``src_bytes`` computed from ``dst``,
example_wrapper.py:131) is not repeated.
"""
from __future__ import annotations

import ctypes
from typing import Optional

from . import _binding

_state = {"sa": None}

_ROPE_LAYOUTS = {"interleaved": 0, "halves": 1}
_ROPE_ARRANGEMENTS = {"own": 0, "shared": 1, "interleaved": 2}
_DTYPE_CODES = {}  # torch dtype -> element type of the C ABI; filled on first use, torch is imported late


def _current_stream(index: int) -> int:
    """The current stream of a device as a pointer (torch.cuda.current_stream without the Stream object: 0.1 us, not 3)."""
    import torch
    return torch._C._cuda_getCurrentRawStream(index)


def _dtype_code(dtype) -> int:
    if not _DTYPE_CODES:
        import torch
        _DTYPE_CODES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    code = _DTYPE_CODES.get(dtype)
    assert code is not None, f"dtype must be float32, bfloat16 or float16, not {dtype}"
    return code


def _below_2_31(*sizes) -> None:
    """The C ABI has 32-bit sizes, and ctypes would cut off what does not fit."""
    assert all(-2 ** 31 <= n < 2 ** 31 for n in sizes), "sizes must be below 2^31"


def _stream_ptr(stream) -> int:
    if stream is None:
        return 0
    if isinstance(stream, int):
        return stream
    if isinstance(stream, ctypes.c_void_p):
        return stream.value or 0
    return int(stream.cuda_stream)


class SideAware:
    """One loaded sideaware.so plus thin, checked wrappers around its launchers."""

    def __init__(self, path: Optional[str] = None):
        self.lib = _binding.load(path)
        self.path = self.lib._path
        self._norm_shapes = {}  # shape and types -> what the C ABI is told of them, and the workspace's size

    # -- errors ---------------------------------------------------------------
    def last_error(self) -> str:
        return (self.lib.sideaware_last_error() or b"").decode()

    def error_count(self) -> int:
        return int(self.lib.sideaware_error_count())

    def _checked(self, before: int, what: str) -> None:
        if self.error_count() != before:
            raise RuntimeError(f"{what}: {self.last_error()}")

    # -- metadata ---------------------------------------------------------------
    def summary(self):
        """(num_sms, num_side0, num_side1, min_sm_per_side, hash_mask)"""
        before = self.error_count()
        out = tuple(self.lib.sideaware_sm_side_summary().contents)
        self._checked(before, "sideaware_sm_side_summary")
        return out

    def summary_dict(self):
        n, s0, s1, m, h = self.summary()
        return {"num_sms": n, "side0": s0, "side1": s1, "min": m, "hash": h}

    def cpu_side_index(self) -> bytes:
        n = self.summary()[0]
        ptr = self.lib.sideaware_cpu_side_index()
        return ctypes.string_at(ptr, n)

    def stats(self) -> dict:
        st = _binding.Stats()
        self.lib.sideaware_get_stats(ctypes.byref(st))
        return st.as_dict()

    def driver_call_times(self) -> dict:
        """Host milliseconds and call counts the allocator spent in driver calls, by kind."""
        ns = (ctypes.c_ulonglong * 8)()
        calls = (ctypes.c_ulonglong * 8)()
        self.lib.sideaware_driver_call_times(ctypes.byref(ns), ctypes.byref(calls))
        names = ["create", "release", "reserve", "map", "unmap", "set_access", "probe", "sync"]
        return {n: {"ms": ns[i] / 1e6, "calls": int(calls[i])} for i, n in enumerate(names)}

    def topology_json(self) -> str:
        return (self.lib.sideaware_topology_json() or b"{}").decode()

    def set_placement(self, mode) -> None:
        modes = {"aware": 0, "unaware": 1, "wrong": 2}
        self.lib.sideaware_set_placement(modes.get(mode, mode))

    # -- raw allocation (no torch) --------------------------------------------
    def malloc(self, size: int, stream=None) -> int:
        p = ctypes.c_void_p()
        rc = self.lib.sideaware_malloc_async(ctypes.byref(p), size, _stream_ptr(stream))
        if rc != 0 or not p.value:
            raise MemoryError(f"sideaware_malloc_async({size}) failed with CUDA error {rc}: {self.last_error()}")
        return int(p.value)

    def free(self, ptr: int, stream=None) -> None:
        rc = self.lib.sideaware_free_async(ptr, _stream_ptr(stream))
        if rc != 0:
            raise RuntimeError(f"sideaware_free_async failed with CUDA error {rc}: {self.last_error()}")

    # -- kernels on raw pointers --------------------------------------------------
    def memcpy_ptr(self, dst: int, src: int, num_bytes: int, device: int = 0, stream=None) -> None:
        before = self.error_count()
        self.lib.sideaware_memcpy(dst, src, num_bytes, device, _stream_ptr(stream))
        self._checked(before, "sideaware_memcpy")

    def rope_backward_ptr(self, dqkv: int, freqs: int, B, T, Nq, Nkv, HS, bf16: bool, device: int = 0, stream=None) -> None:
        _below_2_31(B, T, Nq, Nkv, HS)
        rc = self.lib.sideaware_rope_backward(dqkv, freqs, B, T, Nq, Nkv, HS, 1 if bf16 else 0, device, _stream_ptr(stream))
        if rc != 0:
            raise RuntimeError(f"sideaware_rope_backward failed with CUDA error {rc}: {self.last_error()}")

    def rope_forward_ptr(self, qkv: int, freqs: int, B, T, Nq, Nkv, HS, bf16: bool, device: int = 0, stream=None) -> None:
        _below_2_31(B, T, Nq, Nkv, HS)
        rc = self.lib.sideaware_rope_forward(qkv, freqs, B, T, Nq, Nkv, HS, 1 if bf16 else 0, device, _stream_ptr(stream))
        if rc != 0:
            raise RuntimeError(f"sideaware_rope_forward failed with CUDA error {rc}: {self.last_error()}")

    def rope_precompute_freqs_ptr(self, table: int, dim: int, end: int, theta: float, use_scaled: bool,
                                  device: int = 0, stream=None) -> None:
        _below_2_31(dim, end)
        rc = self.lib.sideaware_rope_precompute_freqs(table, dim, end, theta, 1 if use_scaled else 0, device, _stream_ptr(stream))
        if rc != 0:
            raise RuntimeError(f"sideaware_rope_precompute_freqs failed with CUDA error {rc}: {self.last_error()}")

    def silu_mul_ptr(self, out: int, a: int, b: int, scale: float, n: int, device: int = 0, stream=None) -> None:
        rc = self.lib.sideaware_silu_mul_bf16(out, a, b, scale, n, device, _stream_ptr(stream))
        if rc != 0:
            raise RuntimeError(f"sideaware_silu_mul_bf16 failed with CUDA error {rc}: {self.last_error()}")

    def create_kernel(self, header_code: bytes) -> int:
        if isinstance(header_code, str):
            header_code = header_code.encode()
        return int(self.lib.sideaware_create_kernel(header_code))

    def compile_check(self, header_code: bytes, wide: bool = False) -> str:
        """Compiles a functor header for sm_100a without a GPU; returns "" or the compiler log."""
        if isinstance(header_code, str):
            header_code = header_code.encode()
        buf = ctypes.create_string_buffer(1 << 16)
        rc = self.lib.sideaware_compile_check(header_code, 1 if wide else 0, buf, len(buf))
        log = buf.value.decode()
        if rc == 0:
            if log:  # compiles, but uses something that does not carry over from the reference's launch shape
                import warnings
                warnings.warn(log)
            return ""
        return log or "compile failed"

    def chunk_sides(self, ptr: int, num_bytes: int) -> bytes:
        n = (num_bytes + (ptr & 4095) + 4095) // 4096
        buf = ctypes.create_string_buffer(n)
        got = self.lib.sideaware_chunk_sides(ptr, num_bytes, buf)
        return buf.raw[:got]

    def verify_chunk_sides(self, ptr: int, num_bytes: int, samples: int = 256, seed: int = 0) -> int:
        return int(self.lib.sideaware_verify_chunk_sides(ptr, num_bytes, samples, seed))

    # -- torch tensors --------------------------------------------------------------
    def memcpy(self, dst, src) -> None:
        import torch
        assert dst.device.type == "cuda" and src.device.type == "cuda", "Both tensors must be on CUDA"
        assert dst.dtype == src.dtype, "Source and destination must have the same dtype"
        assert dst.numel() >= src.numel(), "Destination tensor must be at least as large as source"
        assert src.is_contiguous(), "src must be contiguous"
        assert dst.is_contiguous(), "dst must be contiguous"
        assert dst.data_ptr() % 16 == 0 and src.data_ptr() % 16 == 0, "dst and src must be 16-byte aligned"
        self.memcpy_ptr(dst.data_ptr(), src.data_ptr(), src.numel() * src.element_size(),
                        src.device.index, torch.cuda.current_stream(src.device))

    def one_to_one(self, kernel_id: int, dst, src) -> None:
        import torch
        dst_bytes = dst.numel() * dst.element_size() if dst is not None else 0
        src_bytes = src.numel() * src.element_size() if src is not None else 0
        num_bytes = max(src_bytes, dst_bytes)
        assert num_bytes > 0
        for t, name in ((dst, "dst"), (src, "src")):
            assert t is None or (t.is_contiguous() and t.device.type == "cuda"), f"{name} must be contiguous"
        dst_ptr = dst.data_ptr() if dst is not None else 0
        src_ptr = src.data_ptr() if src is not None else 0
        assert dst_ptr % 16 == 0 and src_ptr % 16 == 0, "dst and src must be 16-byte aligned"
        ref = dst if dst is not None else src
        before = self.error_count()
        self.lib.sideaware_one_to_one(kernel_id, num_bytes, dst_ptr, src_ptr, ref.device.index,
                                      _stream_ptr(torch.cuda.current_stream(ref.device)))
        self._checked(before, "sideaware_one_to_one")

    def elementwise(self, kernel_id: int, out0, out1, out2, out3, in0, in1, in2, in3,
                    sideband_tensor=None, sideband_value: int = 0, parallel_chunks: int = 0,
                    forced_sm_per_side: int = 0) -> None:
        import torch
        tensors = [out0, out1, out2, out3, in0, in1, in2, in3]
        names = ["out0", "out1", "out2", "out3", "in0", "in1", "in2", "in3"]
        # num_bytes is the byte size of the one array the kernel moves as 16-byte vectors: in0, or out0 if its
        # element is wider (sideaware.cu:127-129, :1378).  The other arrays may be any size the functor's
        # index function asks for (a short broadcast table, a wider auxiliary array): they do not count.
        num_bytes = max((t.numel() * t.element_size() for t in (in0, out0) if t is not None), default=0)
        assert num_bytes > 0, "in0 or out0 must be given"
        ptrs = []
        for t, name in zip(tensors, names):
            assert t is None or (t.is_contiguous() and t.device.type == "cuda"), f"{name} must be contiguous"
            ptrs.append(t.data_ptr() if t is not None else 0)
            assert ptrs[-1] % 16 == 0, "16B alignment"
        sideband_ptr = sideband_tensor.data_ptr() if sideband_tensor is not None else 0
        ref = next(t for t in tensors if t is not None)
        before = self.error_count()
        self.lib.sideaware_elementwise(kernel_id, num_bytes, *ptrs, sideband_ptr, sideband_value, parallel_chunks,
                                       forced_sm_per_side, ref.device.index,
                                       _stream_ptr(torch.cuda.current_stream(ref.device)))
        self._checked(before, "sideaware_elementwise")

    def rope_forward(self, qkv, freqs_cis, n_q_heads: int, n_kv_heads: int) -> None:
        """In place on packed [B, T, Nq + 2 Nkv, HS] (fp32 or bf16); freqs_cis fp32 [T, HS/2, 2]."""
        import torch
        assert qkv.is_cuda and freqs_cis.is_cuda and qkv.is_contiguous() and freqs_cis.is_contiguous()
        assert qkv.dtype in (torch.float32, torch.bfloat16) and freqs_cis.dtype == torch.float32
        B, T, H, HS = qkv.shape
        assert H == n_q_heads + 2 * n_kv_heads, "head dimension must hold q, k and v heads"
        assert tuple(freqs_cis.shape) == (T, HS // 2, 2), "freqs_cis must be [T, HS/2, 2]"
        self.rope_forward_ptr(qkv.data_ptr(), freqs_cis.data_ptr(), B, T, n_q_heads, n_kv_heads, HS,
                              qkv.dtype == torch.bfloat16, qkv.device.index, torch.cuda.current_stream(qkv.device))

    def rope_backward(self, dqkv, freqs_cis, n_q_heads: int, n_kv_heads: int) -> None:
        """In place on the gradient of a packed [B, T, Nq + 2 Nkv, HS] tensor."""
        import torch
        assert dqkv.is_cuda and freqs_cis.is_cuda and dqkv.is_contiguous() and freqs_cis.is_contiguous()
        assert dqkv.dtype in (torch.float32, torch.bfloat16) and freqs_cis.dtype == torch.float32
        B, T, H, HS = dqkv.shape
        assert H == n_q_heads + 2 * n_kv_heads and tuple(freqs_cis.shape) == (T, HS // 2, 2)
        self.rope_backward_ptr(dqkv.data_ptr(), freqs_cis.data_ptr(), B, T, n_q_heads, n_kv_heads, HS,
                               dqkv.dtype == torch.bfloat16, dqkv.device.index, torch.cuda.current_stream(dqkv.device))

    def rope_precompute_freqs_into(self, freqs_cis, theta: float = 10000.0, use_scaled: bool = False) -> None:
        """Fills an existing fp32 CUDA tensor [end, dim/2, 2] with (cos, sin)."""
        import torch
        assert freqs_cis.is_cuda and freqs_cis.is_contiguous() and freqs_cis.dtype == torch.float32
        assert freqs_cis.dim() == 3 and freqs_cis.shape[2] == 2, "freqs_cis must be [end, dim/2, 2]"
        end, half, _ = freqs_cis.shape
        self.rope_precompute_freqs_ptr(freqs_cis.data_ptr(), 2 * half, end, float(theta), use_scaled,
                                       freqs_cis.device.index, torch.cuda.current_stream(freqs_cis.device))

    def rope_precompute_freqs(self, dim: int, end: int, theta: float = 10000.0, use_scaled: bool = False, device=None):
        """The fp32 table [end, dim/2, 2] of (cos, sin) that rope_forward / rope_backward read, made on the GPU."""
        import torch
        device = torch.device("cuda" if device is None else device)
        assert device.type == "cuda", f"the table is made on a CUDA device, not on {device}"
        table = torch.empty((end, dim // 2, 2), dtype=torch.float32, device=device)
        self.rope_precompute_freqs_ptr(table.data_ptr(), dim, end, float(theta), use_scaled, table.device.index,
                                       torch.cuda.current_stream(table.device))
        return table

    def silu_mul(self, out, a, b, scale: float) -> None:
        import torch
        for t in (out, a, b):
            assert t.is_cuda and t.is_contiguous() and t.dtype == torch.bfloat16
        assert out.numel() == a.numel() == b.numel()
        self.silu_mul_ptr(out.data_ptr(), a.data_ptr(), b.data_ptr(), float(scale), a.numel(), a.device.index,
                          torch.cuda.current_stream(a.device))

    def mxfp8_quantize(self, out, scales, x) -> None:
        """bf16 -> MXFP8 with functors.mxfp8_quantize_bf16: `out` uint8 (E4M3 bytes, one per element), `scales`
        uint8 (E8M0 bytes, one per block of 32 elements; its size must be a multiple of 4), `x` bfloat16.
        A block is reduced inside one warp instruction, which needs x to start on a 64-byte boundary; the
        element count must be a multiple of 8 (whole 16-byte vectors), a last block of fewer than 32
        elements is scaled by the elements it has."""
        import torch
        from . import functors
        assert x.dtype == torch.bfloat16 and out.dtype == torch.uint8 and scales.dtype == torch.uint8
        n = x.numel()
        assert n % 8 == 0, "the element count must be a multiple of 8"
        assert x.data_ptr() % 64 == 0, "x must start on a 64-byte boundary (a block of 32 elements may not straddle two warp instructions)"
        assert out.numel() >= n and scales.numel() >= (n + 31) // 32 and scales.numel() % 4 == 0
        assert n // 8 < 2 ** 31
        kid = self.create_kernel(functors.mxfp8_quantize_bf16())
        # the vector count tells the functor where the last, partial block ends; 0 = there is none (the common case,
        # in which the functor skips that bookkeeping)
        self.elementwise(kid, out[:n], None, None, None, x, None, None, None, scales.view(torch.int32),
                         n // 8 if n % 32 else 0)

    # -- operators of image and video models --------------------------------------
    def _done(self, rc: int, what: str) -> None:
        if rc != 0:
            raise RuntimeError(f"{what} failed with CUDA error {rc}: {self.last_error()}")

    def rope_axes_spectrum(self, pairs_per_axis, theta: float = 10000.0, arrangement: str = "own", device=None):
        """The spectrum that rope_axes_forward / _backward read: int64 [sum(pairs_per_axis)], made on the GPU.
        arrangement "own": every axis has a run of pairs and frequencies theta^(-j/n) of its own; "shared": one series
        theta^(-i/pairs), each axis a run of it; "interleaved": the same series, its pairs dealt to the axes in turn."""
        import torch
        device = torch.device("cuda" if device is None else device)
        assert device.type == "cuda", f"the spectrum is made on a CUDA device, not on {device}"
        index = torch.cuda.current_device() if device.index is None else device.index
        assert arrangement in _ROPE_ARRANGEMENTS, f"arrangement must be one of {sorted(_ROPE_ARRANGEMENTS)}"
        pairs = [int(n) for n in pairs_per_axis]
        assert 1 <= len(pairs) <= 8 and min(pairs) >= 0 and 1 <= sum(pairs) <= 256, "1 to 8 axes and 1 to 256 pairs over all of them"
        spectrum = torch.empty(sum(pairs), dtype=torch.int64, device=device)
        self._done(self.lib.sideaware_rope_axes_spectrum(
            spectrum.data_ptr(), (ctypes.c_int * len(pairs))(*pairs), len(pairs), float(theta), _ROPE_ARRANGEMENTS[arrangement],
            index, _current_stream(index)), "sideaware_rope_axes_spectrum")
        spectrum.rope_axes = len(pairs)  # what the positions are checked against; a copy of the tensor goes without
        return spectrum

    def _rope_axes(self, call, what, qkv, positions, spectrum, n_q_heads, n_kv_heads, layout) -> None:
        import torch
        B, T, H, HS = qkv.shape
        # the C ABI has 32-bit sizes, and ctypes would cut off what does not fit; negative ones are refused as well
        pairs, axes = spectrum.numel(), positions.shape[0]
        assert (B | T | H | HS | n_q_heads | n_kv_heads | pairs | axes) >> 31 == 0, "sizes must be below 2^31"
        assert getattr(spectrum, "rope_axes", axes) == axes, "positions must have the axes that the spectrum was made with"
        device = qkv.get_device()
        assert device >= 0 and positions.get_device() == device and spectrum.get_device() == device, "all tensors must be on one CUDA device"
        assert H == n_q_heads + 2 * n_kv_heads, "head dimension must hold q, k and v heads"
        sb, st, sh, se = qkv.stride()
        assert (se == 1 or HS == 1) and (sh == HS or H <= 1), "heads and their elements must be dense"
        assert positions.dim() == 3 and tuple(positions.shape[1:]) == (B, T), "positions must be [axes, B, T]"
        assert positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64"
        assert spectrum.dim() == 1 and spectrum.dtype == torch.int64 and spectrum.is_contiguous(), "spectrum must be int64 [pairs]"
        assert layout in _ROPE_LAYOUTS, f"layout must be one of {sorted(_ROPE_LAYOUTS)}"
        shape = _binding.RopeAxes(B, T, n_q_heads, n_kv_heads, HS, pairs, axes, _ROPE_LAYOUTS[layout], _dtype_code(qkv.dtype),
                                  1 if positions.dtype == torch.int64 else 0, sb, st, *positions.stride())
        self._done(call(qkv.data_ptr(), positions.data_ptr(), spectrum.data_ptr(), ctypes.byref(shape), device, _current_stream(device)), what)

    def rope_axes_forward(self, qkv, positions, spectrum, n_q_heads: int, n_kv_heads: int, layout: str = "interleaved") -> None:
        """Rotary positions with several axes, in place on packed [B, T, Nq + 2 Nkv, HS] (fp32, bf16 or fp16; any strides
        over B and T): pair i of every q and k head turns by positions[axis of i, b, t] times its frequency.
        positions: int32 or int64 [axes, B, T], any strides and values, with the spectrum's axes (others are refused; where
        the spectrum is a copy that no longer knows them, pairs of axes that the positions lack, and neighbours, become NaN); spectrum:
        rope_axes_spectrum.  A head of which the spectrum's pairs fill only a part keeps its remaining elements.  layout:
        pair i = elements (2i, 2i + 1) ("interleaved") or (i, i + pairs) ("halves")."""
        self._rope_axes(self.lib.sideaware_rope_axes_forward, "sideaware_rope_axes_forward", qkv, positions, spectrum,
                        n_q_heads, n_kv_heads, layout)

    def rope_axes_backward(self, dqkv, positions, spectrum, n_q_heads: int, n_kv_heads: int, layout: str = "interleaved") -> None:
        """In place on the gradient of the packed tensor: the turn by the opposite angle."""
        self._rope_axes(self.lib.sideaware_rope_axes_backward, "sideaware_rope_axes_backward", dqkv, positions, spectrum,
                        n_q_heads, n_kv_heads, layout)

    def _group_norm_shape(self, x, groups, eps, silu, backward, like, stats, params):
        """Checks what forward and backward share; returns (shape for the C ABI, workspace, its size).  `like`: tensors shaped
        as x; `stats`: fp32 [N, groups]; `params`: tensors of C entries, or None."""
        import torch
        size, dtype, device = x.shape, x.dtype, x.get_device()
        assert len(size) >= 2, "x must be a dense CUDA tensor [N, ..., C]"
        N, C = size[0], size[-1]
        # the C ABI has 32-bit sizes (S: 64 bits), and ctypes would cut off what does not fit
        assert (N | C | groups) >> 31 == 0, "samples, channels and groups must be below 2^31"
        assert device >= 0 and x.is_contiguous(), "x must be a dense CUDA tensor [N, ..., C]"
        for t in like:
            assert t.shape == size and t.dtype is dtype and t.is_contiguous() and t.get_device() == device, \
                "out, dx and dout must be dense tensors of x's shape, dtype and device"
        for t in stats:
            assert t.dtype is torch.float32 and t.is_contiguous() and t.numel() == N * groups and t.get_device() == device, \
                "mean and rstd must be dense fp32 [N, groups]"
        param_dtype = None
        for t in params:
            if t is not None:
                assert t.numel() == C and t.is_contiguous() and t.get_device() == device, "weight, bias and their gradients must be dense [C]"
                assert param_dtype is None or t.dtype is param_dtype, "weight, bias and their gradients must have one dtype"
                param_dtype = t.dtype
        key = (size, dtype, groups, eps, silu, backward, param_dtype)
        known = self._norm_shapes.get(key)
        if known is None:
            assert groups >= 1 and C >= 1 and C % groups == 0, "the channels must divide evenly into the groups"
            S = 1
            for n in size[1:-1]:
                S *= n
            shape = _binding.GroupNorm(S, N, C, groups, eps, 1 if silu else 0, _dtype_code(dtype),
                                       0 if param_dtype is None else _dtype_code(param_dtype))
            before = self.error_count()
            need = self.lib.sideaware_group_norm_workspace(ctypes.byref(shape), backward)
            self._checked(before, "sideaware_group_norm_workspace")
            if len(self._norm_shapes) >= 256:  # a program whose shapes never come back
                self._norm_shapes.clear()
            known = self._norm_shapes[key] = (shape, need)
        shape, need = known
        return shape, (torch.empty(need, dtype=torch.uint8, device=x.device) if need else None), need

    def group_norm_forward(self, out, mean, rstd, x, weight, bias, groups: int, eps: float = 1e-5, silu: bool = True) -> None:
        """Group norm, then SiLU unless silu is False, on dense channels-last x [N, ..., C] (fp32, bf16 or fp16; a
        channels_last [N, C, H, W] tensor is passed as x.permute(0, 2, 3, 1)).  out: like x, may be x.  mean and rstd:
        fp32 [N, groups], written for the backward pass.  weight, bias: [C] of one dtype, each may be None."""
        shape, workspace, size = self._group_norm_shape(x, groups, eps, silu, 0, (out,), (mean, rstd), (weight, bias))
        device = x.get_device()
        self._done(self.lib.sideaware_group_norm_forward(
            out.data_ptr(), mean.data_ptr(), rstd.data_ptr(), x.data_ptr(), weight.data_ptr() if weight is not None else 0,
            bias.data_ptr() if bias is not None else 0, ctypes.byref(shape), workspace.data_ptr() if size else 0, size,
            device, _current_stream(device)), "sideaware_group_norm_forward")

    def group_norm_backward(self, dx, dweight, dbias, dout, x, mean, rstd, weight, bias, groups: int, silu: bool = True) -> None:
        """Gradients of group_norm_forward: dx like x (may be dout or x), dweight and dbias [C] like weight and bias, each
        may be None.  mean and rstd: the forward pass's."""
        shape, workspace, size = self._group_norm_shape(x, groups, 0.0, silu, 1, (dx, dout), (mean, rstd), (weight, bias, dweight, dbias))
        device = x.get_device()
        ptr = [t.data_ptr() if t is not None else 0 for t in (dx, dweight, dbias, dout, x, mean, rstd, weight, bias)]
        self._done(self.lib.sideaware_group_norm_backward(
            *ptr, ctypes.byref(shape), workspace.data_ptr() if size else 0, size, device, _current_stream(device)),
            "sideaware_group_norm_backward")

    def _dropout_check(self, out, x, rng, residual) -> int:
        import torch
        device = x.get_device()
        assert device >= 0 and x.is_contiguous(), "x must be a dense CUDA tensor"
        for t in (out, residual):
            assert t is None or (t.shape == x.shape and t.dtype is x.dtype and t.is_contiguous() and t.get_device() == device), \
                "out and residual must be dense tensors of x's shape, dtype and device"
        assert rng.dtype is torch.int64 and rng.numel() == 2 and rng.is_contiguous() and rng.get_device() == device, \
            "rng must be int64 (seed, number of the call) on x's device"
        return device

    def dropout_forward(self, out, x, rng, p: float, residual=None) -> None:
        """out = residual + (keep ? x / (1 - p) : 0) (fp32, bf16 or fp16; out may be x or residual).  The mask is drawn
        from rng, an int64 CUDA tensor (seed, number of the call): every call of a model takes a number of its own, and
        dropout_backward the forward pass's pair.  The pair is read on the device, so a replayed CUDA graph that advances
        it draws new masks."""
        device = self._dropout_check(out, x, rng, residual)
        self._done(self.lib.sideaware_dropout_forward(
            out.data_ptr(), x.data_ptr(), residual.data_ptr() if residual is not None else 0, rng.data_ptr(), p, x.numel(),
            _dtype_code(x.dtype), device, _current_stream(device)), "sideaware_dropout_forward")

    def dropout_backward(self, dx, dout, rng, p: float) -> None:
        """dx = keep ? dout / (1 - p) : 0 with the forward pass's rng (the residual's gradient is dout itself)."""
        device = self._dropout_check(dx, dout, rng, None)
        self._done(self.lib.sideaware_dropout_backward(
            dx.data_ptr(), dout.data_ptr(), rng.data_ptr(), p, dout.numel(), _dtype_code(dout.dtype), device,
            _current_stream(device)), "sideaware_dropout_backward")

    def side_index_tensor(self):
        import torch
        n = self.summary()[0]
        t = torch.zeros(n, dtype=torch.uint8, device="cuda")
        self.lib.sideaware_fill_side_index(t.data_ptr())
        return t

    # -- torch integration -----------------------------------------------------------
    def install_allocator(self) -> None:
        """Routes torch's CUDA allocations through sideaware_malloc_auto / sideaware_free_auto
        (test.py:14-15).  Must run before the first CUDA allocation of the process."""
        import torch
        alloc = torch.cuda.memory.CUDAPluggableAllocator(self.path, "sideaware_malloc_auto", "sideaware_free_auto")
        torch.cuda.memory.change_current_allocator(alloc)

    def register_ops(self) -> None:
        """torch.ops.sideaware.{memcpy, one_to_one, elementwise, rope_forward, silu_mul}"""
        from . import torch_ops
        torch_ops.register(self)


# ---------------------------------------------------------------------------
# module-level functions with the reference wrapper's names (example_wrapper.py:21-43)
# ---------------------------------------------------------------------------
def sideaware_init(path: Optional[str] = None, install_allocator: bool = True) -> SideAware:
    sa = SideAware(path)
    if install_allocator:
        sa.install_allocator()
    sa.register_ops()
    _state["sa"] = sa
    _state["info"] = sa.summary()
    _state["torch_side_index"] = sa.side_index_tensor()
    print(f"L2 Side Aware metadata: {sa.summary_dict()}")
    return sa


def sideaware_enabled() -> int:
    return 1 if _state["sa"] is not None else 0


def _sa() -> SideAware:
    if _state["sa"] is None:
        raise RuntimeError("call sideaware_init() first")
    return _state["sa"]


def sideaware_create_kernel(header_code: bytes) -> int:
    return _sa().create_kernel(header_code)


def sideaware_torch_side_index():
    return _state.get("torch_side_index")


def sideaware_gpu_side_index():
    return _sa().lib.sideaware_gpu_side_index()


def sideaware_cpu_side_index():
    return _sa().lib.sideaware_cpu_side_index()


def sideaware_info():
    n, s0, s1, m, h = _state.get("info", (0, 0, 0, 0, 0))
    return {"num_sms": n, "side0": s0, "side1": s1, "min": m, "hash": h}


def sideaware_info_raw():
    return _state.get("info", (0, 0, 0, 0, 0))
