"""Attention over whole prompts, and what a prompt hands to the cache: the side of the path before the first decode step.

``prompt_attention`` computes what the reference's prefill leaves to a flash-attention library (model/llama_hqe.py:141-166), for
packed sequences of any lengths in one call; ``prompt_importance`` the head-summed probabilities of each sequence's last queries,
which seed the importance ring (:124, 141-166; model/public_func.py:247-252).  Both are hand-written kernels of libhqkv
(hqekv_b200/csrc/prompt.cu).  They have no backward pass, like every operator of this package, and refuse inputs that need one.

Layout: tokens x heads x channels, the tokens of all sequences one behind another.  ``seq_starts`` (int32 or int64, ``n + 1`` entries on
the tensors' device) says where each sequence begins and the last one ends.  They do not decrease; what lies outside of the tokens is taken
as the nearest end of them.  A padded batch ``[B, heads, S, 128]`` is packed as
``x.transpose(1, 2).reshape(B * S, heads, 128)`` with starts ``0, S, 2 S, ...`` - a view where the batch is stored token by token.
"""
import ctypes as C

import torch
from torch.autograd import forward_ad

from ._lib import Prompt, check, host, lib, ptr, require_cuda, stream_ptr

HEAD_DIM = 128
MAX_ROWS = 64   # HQKV_IMPORTANCE_ROWS
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def usable(x):
    """Whether the kernels read a [tokens, heads, 128] tensor where it is."""
    return x.stride(2) == 1 and x.data_ptr() % 16 == 0 and all(x.shape[d] < 2 or (x.stride(d) > 0 and x.stride(d) % 8 == 0) for d in (0, 1))


def no_gradient(*tensors):
    """Refuse what derivatives are asked of (of a dual tensor under no_grad, too: that does not end forward mode)."""
    for x in tensors:
        if x is None:
            continue
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("these operators have no backward pass: call them under torch.no_grad()")
        if forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("these operators have no forward derivatives: unpack dual tensors before the call")


def _tensor(name, x, like=None, heads=None, tokens=None):
    """A [tokens, heads, 128] operand as the kernels take it: channels adjacent, 16-byte aligned rows (copied where it is not)."""
    if x.dim() != 3 or x.shape[2] != HEAD_DIM:
        raise ValueError(f"{name} must be [tokens, heads, {HEAD_DIM}] (got {tuple(x.shape)})")
    if like is not None and (x.dtype != like.dtype or x.device != like.device):
        raise ValueError(f"{name} must have the type and device of q")
    if heads is not None and x.shape[1] != heads:
        raise ValueError(f"{name} must have {heads} heads (got {x.shape[1]})")
    if tokens is not None and x.shape[0] != tokens:
        raise ValueError(f"{name} must have {tokens} tokens (got {x.shape[0]})")
    no_gradient(x)
    return x if usable(x) else x.clone(memory_format=torch.contiguous_format)


def _starts(name, x, device, n=None):
    if not torch.is_tensor(x) or x.dim() != 1 or x.numel() < 1 or x.dtype not in (torch.int32, torch.int64) or x.device != device:
        raise ValueError(f"{name} must be a 1-D int32 or int64 tensor on the device of q")
    if n is not None and x.numel() != n:
        raise ValueError(f"{name} must have {n} entries like seq_starts (got {x.numel()})")
    if x.dtype == torch.int64:   # (starts out of range are taken as the nearest, also those that int32 does not hold)
        x = x.clamp(-1, 2 ** 31 - 1)
    return x.to(torch.int32).contiguous()


def _describe(q, k, v, seq_starts, kv_starts, prefix, causal, scale):
    """(descriptor, tensors it points into) after all checks."""
    if q.dtype not in _DTYPES:
        raise ValueError("q must be float16 or bfloat16")
    q = _tensor("q", q)
    k = _tensor("k", k, q)
    nh, nkv = q.shape[1], k.shape[1]
    if nh == 0 or nkv == 0 or nh % nkv:
        raise ValueError(f"q must have a multiple of k's heads (got {nh} and {nkv})")
    if v is not None:
        v = _tensor("v", v, q, nkv, k.shape[0])
    seq_starts = _starts("seq_starts", seq_starts, q.device)
    if kv_starts is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError("k must have as many tokens as q where kv_starts is not given")
        kv_starts = seq_starts
    else:
        kv_starts = _starts("kv_starts", kv_starts, q.device, seq_starts.numel())
    scale = C.c_float(HEAD_DIM ** -0.5 if scale is None else scale).value   # as the kernels take it
    if not 0.0 < scale < 1e38:
        raise ValueError("scale must be positive, and below 1e38")
    p = Prompt()
    p.dtype, p.D, p.nh_q, p.nh_kv = _DTYPES[q.dtype], HEAD_DIM, nh, nkv
    p.n_seqs, p.causal, p.scale = seq_starts.numel() - 1, int(bool(causal)), scale
    p.total_q, p.total_k = q.shape[0], k.shape[0]
    p.q, p.q_token, p.q_head = ptr(q), q.stride(0), q.stride(1)
    p.k, p.k_token, p.k_head = ptr(k), k.stride(0), k.stride(1)
    if v is not None:
        p.v, p.v_token, p.v_head = ptr(v), v.stride(0), v.stride(1)
    p.q_starts, p.k_starts = ptr(seq_starts), ptr(kv_starts)
    keep = [q, k, v, seq_starts, kv_starts]
    if prefix is not None:
        pk, pv = prefix
        pk = _tensor("the prefix's k", pk, q, nkv)
        pv = _tensor("the prefix's v", pv, q, nkv, pk.shape[0])
        p.prefix_len = pk.shape[0]
        p.prefix_k, p.prefix_k_token, p.prefix_k_head = ptr(pk), pk.stride(0), pk.stride(1)
        p.prefix_v, p.prefix_v_token, p.prefix_v_head = ptr(pv), pv.stride(0), pv.stride(1)
        keep += [pk, pv]
    require_cuda(*keep)
    return p, keep


def prompt_attention(q, k, v, seq_starts, kv_starts=None, *, prefix=None, causal=True, scale=None, out=None):
    """softmax(scale q K^T) V over packed sequences -> (out [Tq, nh_q, 128] of q's type, lse float32 [nh_q, Tq]).

    q [Tq, nh_q, 128], k and v [Tk, nh_kv, 128], float16 or bfloat16, any strides with adjacent channels; nh_q a multiple of nh_kv
    (query heads of one kv head are neighbours).  ``kv_starts``: where the keys of each sequence begin, if they are not those of
    the queries; a causal query sees its own keys up to its distance from the end (query i of Lq sees keys j <= i + Lk - Lq), so a
    chunk of a prompt attends to all that is cached before it.  ``prefix`` = (k, v) [P, nh_kv, 128]: tokens that every query of every
    sequence sees before its own keys.  ``scale``: 1 / sqrt(128) if not given.  ``out``: a contiguous, 32-byte aligned tensor to write to, other memory than the inputs'.

    ``lse`` is the natural logarithm of each row's softmax denominator.  A query that sees no key has output 0 and lse -inf.
    Rows of queries in no sequence (behind the last start, or before the first) are not written: in ``out`` they stay as they were,
    in results allocated here they are undefined.  What a query does not see has no influence on its output, whatever it holds.  Probabilities are
    rounded to the type of v before the product with it; sums, maxima and the output's accumulator are fp32."""
    if out is None:
        pk, pv = prefix or (None, None)
        done = host.prompt_attention(q, k, v, seq_starts, kv_starts, pk, pv, causal, scale)
        if done is not None:
            return done
    # what the native path does not take as it is: operands to be copied, and everything that is an error
    no_gradient(out)
    p, keep = _describe(q, k, v, seq_starts, kv_starts, prefix, causal, scale)
    q = keep[0]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() or out.data_ptr() % 32:
        raise ValueError("out must be a contiguous, 32-byte aligned tensor of q's shape, type and device")
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        need = lib.hqkv_prompt_workspace_bytes(C.byref(p))
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        check(lib.hqkv_prompt_attention(C.byref(p), ptr(out), ptr(lse), ptr(scratch), need, stream_ptr(q.device)))
    return out, lse


def prompt_importance(q, k, lse, seq_starts, kv_starts=None, *, rows=20, causal=True, scale=None, out=None):
    """Head-summed probabilities of each sequence's last ``rows`` queries -> float16 [rows, Tk].

    Row r holds, for every key of a sequence, what the r-th of the sequence's last t = min(rows, Lq) queries gives it, summed over
    the query heads in fp32 and rounded once; rows r >= t are 0 (a ring is seeded with the first t), and so are keys that the query
    does not see.  ``lse`` [nh_q, Tq] as
    ``prompt_attention`` returned it for the same q and keys; only those queries' entries are read.  (With a prefix the rows of a head add up to 1
    minus the prefix's share.)  ``rows``: 1 to 64.  Columns of keys in no sequence are not written: in ``out`` they stay as they were, in
    a result allocated here they are undefined."""
    if isinstance(rows, bool) or not isinstance(rows, int) or not 1 <= rows <= MAX_ROWS:
        raise ValueError(f"rows must be an integer from 1 to {MAX_ROWS}")
    if out is None:
        done = host.prompt_importance(q, k, None, seq_starts, kv_starts, None, None, causal, scale, lse, rows)
        if done is not None:
            return done
    no_gradient(lse, out)
    p, keep = _describe(q, k, None, seq_starts, kv_starts, None, causal, scale)
    q, k = keep[0], keep[1]
    if lse.shape != (q.shape[1], q.shape[0]) or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError("lse must be float32 [nh_q, Tq] on the device of q")
    lse = lse.contiguous()
    if out is None:
        out = torch.empty(rows, k.shape[0], dtype=torch.float16, device=q.device)
    elif out.shape != (rows, k.shape[0]) or out.dtype != torch.float16 or out.device != q.device or not out.is_contiguous():
        raise ValueError("out must be a contiguous float16 [rows, Tk] tensor on the device of q")
    with torch.cuda.device(q.device):
        check(lib.hqkv_prompt_importance(C.byref(p), ptr(lse), rows, ptr(out), stream_ptr(q.device)))
    return out


def waits_expired(device=None, *, reset=False):
    """How many CTAs of these kernels have given up waiting for their own copies and products on ``device`` (the current one if not
    given) since the library was loaded or the count was last ``reset``: 0 unless the GPU is not working properly.  What such a CTA should have
    written stays as it was, and no call can say so when it returns, since it does not wait for the GPU: a program that wants to know
    asks here, which does wait.  Not for calls that are being captured."""
    count = C.c_uint()
    with torch.cuda.device(device):
        check(lib.hqkv_prompt_waits_expired(int(bool(reset)), C.byref(count)))
    return count.value
