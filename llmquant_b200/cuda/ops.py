import ctypes

import torch
import torch.nn.functional as F

from llmquant_b200 import native
from llmquant_b200.cuda.build import load_extension


def fake_quantize_cuda(x: torch.Tensor, args, return_scale: bool = False):
    """Quant-dequant on the GPU, bit-exact with the reference's `fake_quantize`.

    Same contract as llmquant/cuda/ops.py:8-29: groups run along the last axis, "channel" and
    "token" are the one-group case, and a last axis that is not a whole number of groups is
    zero-padded for the kernel and trimmed afterwards (a zero cannot move an abs-max).
    """
    if args.strategy == "group":
        group_size = args.group_size
    elif args.strategy in ("channel", "token"):
        group_size = x.shape[-1]
    else:
        raise ValueError(f"unsupported strategy {args.strategy!r}")
    width = x.shape[-1]
    tail = width % group_size
    padded = F.pad(x, (0, group_size - tail)) if tail else x
    out, scale = load_extension().fake_quant_group(padded, args.num_bits, group_size, return_scale)
    if tail:
        out = out[..., :width]
    return (out, scale) if return_scale else out


def check_rope_tables(cos, sin, device, head_dim):
    """The rotated width of fp32 angle tables [table_len, rot / 2] on `device`."""
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise RuntimeError("cos and sin must be float32 tables of one shape [positions, rotated / 2]")
    if cos.device != device or sin.device != device or not (cos.is_contiguous() and sin.is_contiguous()):
        raise RuntimeError(f"cos and sin must be contiguous on {device}")
    rot = 2 * cos.shape[1]
    if rot == 0 or rot > head_dim or rot % 16:
        raise RuntimeError(f"the tables turn {rot} values: a multiple of 16 up to head_dim {head_dim} is needed")
    return rot


def check_norm_weights(q_weight, k_weight, dtype, device, head_dim):
    if (q_weight is None) != (k_weight is None):
        raise RuntimeError("norm weights are given for both queries and keys or for neither")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype != dtype or w.device != device or w.shape != (head_dim,) or not w.is_contiguous()):
            raise RuntimeError(f"a norm weight must be a contiguous {dtype} [{head_dim}] on {device}")


def qk_norm_rope(q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, out=None):
    """Norms of queries and keys for each head and the position rotation, in one launch.

    q [B, T, Hq, D] and k [B, T, Hk, D] (any strides with D contiguous, e.g. slices of the fused
    projection's output; float32, float16 or bfloat16), cos / sin float32 [positions, rot / 2],
    positions int64 [B, T] (or expandable to it). Returns new (q, k), or writes `out` = (q, k),
    which may be the inputs themselves. Weights [D] of q's dtype, both None for a model without
    these norms. fp32 inside, one rounding. No gradient."""
    if not (q.is_cuda and k.is_cuda):
        raise RuntimeError("q and k must be CUDA tensors")
    if q.dtype not in native.DTYPE_ID:
        raise RuntimeError(f"q must be float32, float16 or bfloat16, got {q.dtype}")
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise RuntimeError(f"q and k must be [batch, tokens, heads, head_dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    if k.dtype != q.dtype or k.device != q.device:
        raise RuntimeError("q and k must share dtype and device")
    batch, tokens, heads, dim = q.shape
    if dim % 8 or not 16 <= dim <= 256:
        raise RuntimeError(f"head_dim must be a multiple of 8 in [16, 256], got {dim}")
    rot = check_rope_tables(cos, sin, q.device, dim)
    check_norm_weights(q_weight, k_weight, q.dtype, q.device, dim)
    if positions.dtype != torch.int64 or positions.device != q.device:
        raise RuntimeError(f"positions must be int64 on {q.device}")
    positions = positions.expand(batch, tokens)
    if q.stride(3) != 1:
        q = q.contiguous()
    if k.stride(3) != 1:
        k = k.contiguous()
    if out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    else:
        q_out, k_out = out
        for t, like in ((q_out, q), (k_out, k)):
            if t.shape != like.shape or t.dtype != q.dtype or t.device != q.device or t.stride(3) != 1:
                raise RuntimeError("out must hold tensors of the inputs' shape, dtype and device, head_dim contiguous")
    if q.numel() + k.numel() == 0:
        return q_out, k_out
    strides = [(ctypes.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, q_out, k_out)]
    with torch.cuda.device(q.device):
        native.call("lq_qk_norm_rope", q.data_ptr(), k.data_ptr(), strides[0], strides[1], q_out.data_ptr(),
                    k_out.data_ptr(), strides[2], strides[3], native.DTYPE_ID[q.dtype], batch, tokens, heads,
                    k.shape[2], dim, native.ptr(q_weight), native.ptr(k_weight), eps, cos.data_ptr(), sin.data_ptr(),
                    cos.shape[0], rot, int(interleaved), positions.data_ptr(), positions.stride(0),
                    positions.stride(1), 1, native.stream_ptr(q.device))
    return q_out, k_out
