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
    shape = cos.shape
    if len(shape) != 2 or shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise RuntimeError("cos and sin must be float32 tables of one shape [positions, rotated / 2]")
    if cos.device != device or sin.device != device or not (cos.is_contiguous() and sin.is_contiguous()):
        raise RuntimeError(f"cos and sin must be contiguous on {device}")
    rot = 2 * shape[1]
    if rot == 0 or rot > head_dim or rot % 16 or shape[0] == 0:
        raise RuntimeError(f"the tables turn {rot} values: a multiple of 16 up to head_dim {head_dim} is needed")
    return shape[0], rot


def check_norm_weights(q_weight, k_weight, dtype, device, head_dim):
    """Their addresses (0: no norms)."""
    if q_weight is None and k_weight is None:
        return 0, 0
    if q_weight is None or k_weight is None:
        raise RuntimeError("norm weights are given for both queries and keys or for neither")
    for w in (q_weight, k_weight):
        if w.dtype is not dtype or w.device != device or w.shape != (head_dim,) or not w.is_contiguous():
            raise RuntimeError(f"a norm weight must be a contiguous {dtype} [{head_dim}] on {device}")
    return q_weight.data_ptr(), k_weight.data_ptr()


def qk_norm_rope(q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, out=None):
    """Norms of queries and keys for each head and the position rotation, in one launch.

    q [B, T, Hq, D] and k [B, T, Hk, D] (any strides with D contiguous, e.g. slices of the fused
    projection's output; float32, float16 or bfloat16), cos / sin float32 [positions, rot / 2],
    positions int64 [B, T] (or expandable to it). Returns new (q, k), or writes `out` = (q, k),
    which may be the inputs themselves (but not overlap them otherwise). Weights [D] of q's dtype,
    both None for a model without these norms. fp32 inside, one rounding. A position outside the
    tables gives NaN. No gradient."""
    device, dtype, shape, k_shape = q.device, q.dtype, q.shape, k.shape
    if device.type != "cuda" or k.device != device:
        raise RuntimeError("q and k must be CUDA tensors of one device")
    if dtype not in native.DTYPE_ID:
        raise RuntimeError(f"q must be float32, float16 or bfloat16, got {dtype}")
    if k.dtype is not dtype:
        raise RuntimeError(f"q and k must share a dtype, got {dtype} and {k.dtype}")
    if len(shape) != 4 or len(k_shape) != 4 or shape[:2] != k_shape[:2] or shape[3] != k_shape[3]:
        raise RuntimeError(f"q and k must be [batch, tokens, heads, head_dim], got {tuple(shape)} and {tuple(k_shape)}")
    batch, tokens, heads, dim = shape
    if dim % 8 or not 16 <= dim <= 256:
        raise RuntimeError(f"head_dim must be a multiple of 8 in [16, 256], got {dim}")
    table_len, rot = check_rope_tables(cos, sin, device, dim)
    wq, wk = check_norm_weights(q_weight, k_weight, dtype, device, dim)
    if positions.dtype is not torch.int64 or positions.device != device:
        raise RuntimeError(f"positions must be int64 on {device}")
    if positions.shape != shape[:2]:
        positions = positions.expand(batch, tokens)
    qs, ks = q.stride(), k.stride()
    if qs[3] != 1:
        q = q.contiguous()
        qs = q.stride()
    if ks[3] != 1:
        k = k.contiguous()
        ks = k.stride()
    if out is None:
        q_out, k_out = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k))
    else:
        q_out, k_out = out
        for t, like in ((q_out, shape), (k_out, k_shape)):
            if t.shape != like or t.dtype is not dtype or t.device != device or t.stride(3) != 1:
                raise RuntimeError("out must hold tensors of the inputs' shape, dtype and device, head_dim contiguous")
    if q_out.numel() + k_out.numel() == 0:
        return q_out, k_out
    native.launch("lq_qk_norm_rope", device.index, q.data_ptr(), k.data_ptr(), native.int64s(qs), native.int64s(ks),
                  q_out.data_ptr(), k_out.data_ptr(), native.int64s(q_out.stride()), native.int64s(k_out.stride()),
                  native.DTYPE_ID[dtype], batch, tokens, heads, k_shape[2], dim, wq, wk, eps, cos.data_ptr(),
                  sin.data_ptr(), table_len, rot, int(interleaved), positions.data_ptr(), *positions.stride(), 1)
    return q_out, k_out
