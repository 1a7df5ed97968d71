"""torch.ops.sideaware.* registration (the custom ops of test.py:147-157, plus rope_forward,
rope_backward, rope_freqs, silu_mul and the operators of image and video models).  Kept in a module of its own WITHOUT postponed annotation evaluation:
torch.library.infer_schema reads the real annotation objects."""
from typing import Optional

import torch
from torch import Tensor

_registered = {}


def register(sa) -> None:
    """Registers the ops once per process, bound to the loaded library `sa`."""
    if _registered:
        return

    def memcpy(dst: Tensor, src: Tensor) -> None:
        sa.memcpy(dst, src)

    def one_to_one(kernel_id: int, dst: Tensor, src: Tensor) -> None:
        sa.one_to_one(kernel_id, dst, src)

    def elementwise(kernel_id: int, out0: Tensor, out1: Optional[Tensor], out2: Optional[Tensor],
                    out3: Optional[Tensor], in0: Optional[Tensor], in1: Optional[Tensor], in2: Optional[Tensor],
                    in3: Optional[Tensor], sideband_tensor: Optional[Tensor] = None, sideband_value: int = 0,
                    parallel_chunks: int = 0, forced_sm_per_side: int = 0) -> None:
        sa.elementwise(kernel_id, out0, out1, out2, out3, in0, in1, in2, in3, sideband_tensor, sideband_value,
                       parallel_chunks, forced_sm_per_side)

    def rope_forward(qkv: Tensor, freqs_cis: Tensor, n_q_heads: int, n_kv_heads: int) -> None:
        sa.rope_forward(qkv, freqs_cis, n_q_heads, n_kv_heads)

    def rope_backward(dqkv: Tensor, freqs_cis: Tensor, n_q_heads: int, n_kv_heads: int) -> None:
        sa.rope_backward(dqkv, freqs_cis, n_q_heads, n_kv_heads)

    def rope_freqs(freqs_cis: Tensor, theta: float, use_scaled: bool) -> None:
        sa.rope_precompute_freqs_into(freqs_cis, theta, use_scaled)

    def silu_mul(out: Tensor, a: Tensor, b: Tensor, scale: float) -> None:
        sa.silu_mul(out, a, b, scale)

    def rope_axes_forward(qkv: Tensor, positions: Tensor, spectrum: Tensor, n_q_heads: int, n_kv_heads: int,
                          layout: str = "interleaved") -> None:
        sa.rope_axes_forward(qkv, positions, spectrum, n_q_heads, n_kv_heads, layout)

    def rope_axes_backward(dqkv: Tensor, positions: Tensor, spectrum: Tensor, n_q_heads: int, n_kv_heads: int,
                           layout: str = "interleaved") -> None:
        sa.rope_axes_backward(dqkv, positions, spectrum, n_q_heads, n_kv_heads, layout)

    def group_norm_forward(out: Tensor, mean: Tensor, rstd: Tensor, x: Tensor, weight: Optional[Tensor],
                           bias: Optional[Tensor], groups: int, eps: float = 1e-5, silu: bool = True) -> None:
        sa.group_norm_forward(out, mean, rstd, x, weight, bias, groups, eps, silu)

    def group_norm_backward(dx: Tensor, dweight: Optional[Tensor], dbias: Optional[Tensor], dout: Tensor, x: Tensor,
                            mean: Tensor, rstd: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int,
                            silu: bool = True) -> None:
        sa.group_norm_backward(dx, dweight, dbias, dout, x, mean, rstd, weight, bias, groups, silu)

    def dropout_forward(out: Tensor, x: Tensor, rng: Tensor, p: float, residual: Optional[Tensor] = None) -> None:
        sa.dropout_forward(out, x, rng, p, residual)

    def dropout_backward(dx: Tensor, dout: Tensor, rng: Tensor, p: float) -> None:
        sa.dropout_backward(dx, dout, rng, p)

    lib = torch.library.Library("sideaware", "FRAGMENT")

    def reg(name, fn, mutates):
        schema = torch.library.infer_schema(fn, mutates_args=mutates)
        lib.define(name + schema)
        lib.impl(name, fn, "CUDA")

    reg("memcpy", memcpy, ["dst"])
    reg("one_to_one", one_to_one, ["dst"])
    reg("elementwise", elementwise, ["out0", "out1", "out2", "out3", "sideband_tensor"])
    reg("rope_forward", rope_forward, ["qkv"])
    reg("rope_backward", rope_backward, ["dqkv"])
    reg("rope_freqs", rope_freqs, ["freqs_cis"])
    reg("silu_mul", silu_mul, ["out"])
    reg("rope_axes_forward", rope_axes_forward, ["qkv"])
    reg("rope_axes_backward", rope_axes_backward, ["dqkv"])
    reg("group_norm_forward", group_norm_forward, ["out", "mean", "rstd"])
    reg("group_norm_backward", group_norm_backward, ["dx", "dweight", "dbias"])
    reg("dropout_forward", dropout_forward, ["out"])
    reg("dropout_backward", dropout_backward, ["dx"])
    _registered["lib"] = lib
