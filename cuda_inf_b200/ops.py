"""Operators of the reference's decode path on torch CUDA tensors.

Names and argument meaning follow the kernels of src/engine.cu in
g023/cuda_inf (gemv_int4, rmsnorm, rope, kv_commit_group, ...); each call goes
through the C ABI of libcuinf.so on the current torch CUDA stream.  Tensors
must be CUDA and contiguous (the serving operators at the end also take
strided token rows, and run on their tensors' device); fp16 activations, u8 packed INT4 / FP8, fp32
GEMV outputs.  Errors raise CuinfError; nothing falls back to the CPU.
"""
import ctypes
import functools

import torch

from ._lib import check, lib

__all__ = [
    "gemv_int4", "gemv_fp16", "rmsnorm", "rmsnorm_head", "rope", "kv_write_tail",
    "kv_commit_group", "attn_decode", "attn_decode_noalloc", "conv_pre", "conv_apply", "conv_update_state", "swiglu",
    "acc_scaled", "add_inplace", "add_f32_inplace", "f32_to_f16", "embed_gather", "argmax",
    "moe_route", "moe_ffn", "quantize_int4", "expert_table",
    "attn_varlen", "kv_paged_append", "attn_paged", "paged_error",
]


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return ctypes.c_void_p(t.data_ptr())


def _dt(t, dtype, name):
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def gemv_int4(x, packed, scales, y=None):
    """y[m,n] = sum_k x[m,k] * (nib-8) * scale[n,k/128]  (gemv_int4, engine.cu:83-109).

    x fp16 [M,K] (or [K]); packed u8 [N,K/2]; scales fp16 [N,K/128]; y fp32 [M,N]."""
    _dt(x, torch.float16, "x"), _dt(packed, torch.uint8, "packed"), _dt(scales, torch.float16, "scales")
    N, K = packed.shape[0], packed.shape[1] * 2
    M = x.numel() // K
    if y is None:
        y = torch.empty((M, N) if x.dim() > 1 else (N,), dtype=torch.float32, device=x.device)
    check(lib().cuinf_gemv_int4(_p(x), _p(packed), _p(scales), _p(y), M, N, K, _stream()))
    return y


def gemm_int4_tc(x, packed, scales, y=None):
    """Tensor-core form of gemv_int4 for M activation rows (tcgen05)."""
    _dt(x, torch.float16, "x"), _dt(packed, torch.uint8, "packed"), _dt(scales, torch.float16, "scales")
    N, K = packed.shape[0], packed.shape[1] * 2
    M = x.numel() // K
    if y is None:
        y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    check(lib().cuinf_gemm_int4_tc(_p(x), _p(packed), _p(scales), _p(y), M, N, K, _stream()))
    return y


def gemm_fp16_tc(x, W, want_logits=True):
    """Tensor-core x[M,K] . W[N,K]^T with the fused argmax; returns
    (logits fp32 [M,N] or None, argmax int [M])."""
    _dt(x, torch.float16, "x"), _dt(W, torch.float16, "W")
    N, K = W.shape
    M = x.numel() // K
    y = torch.empty((M, N), dtype=torch.float32, device=x.device) if want_logits else None
    keys = torch.zeros(M, dtype=torch.int64, device=x.device)
    check(lib().cuinf_gemm_fp16_tc(_p(x), _p(W), _p(y) if y is not None else None, M, N, K, _p(keys),
                                   _stream()))
    idx = [lib().cuinf_argmax_key_index(int(k) & 0xFFFFFFFFFFFFFFFF) for k in keys.cpu().tolist()]
    return y, idx


def gemv_fp16(x, W, y=None):
    """y[m,n] = sum_k x[m,k] * W[n,k]  (gemv_fp16, engine.cu:112-128)."""
    _dt(x, torch.float16, "x"), _dt(W, torch.float16, "W")
    N, K = W.shape
    M = x.numel() // K
    if y is None:
        y = torch.empty((M, N) if x.dim() > 1 else (N,), dtype=torch.float32, device=x.device)
    check(lib().cuinf_gemv_fp16(_p(x), _p(W), _p(y), M, N, K, _stream()))
    return y


def rmsnorm(inp, w, out=None, eps=1e-5):
    """half(x * rsqrt(mean(x^2) + eps) * w) per row  (rmsnorm, engine.cu:131-144)."""
    D = w.numel()
    M = inp.numel() // D
    if out is None:
        out = torch.empty_like(inp)
    check(lib().cuinf_rmsnorm(_p(inp), _p(w), _p(out), M, D, eps, _stream()))
    return out


def rmsnorm_head(inp, w, out=None, eps=1e-5):
    """Per-head RMSNorm over head_dim 64  (rmsnorm_head, engine.cu:148-158)."""
    return rmsnorm(inp, w, out, eps)


def rope(q, k, pos, theta=5e6):
    """In-place NEOX RoPE on q [S,nq,64] and k [S,nk,64]  (rope, engine.cu:161-182)."""
    S = pos.numel()
    nq = q.numel() // (S * 64)
    nk = k.numel() // (S * 64) if k is not None else 0
    check(lib().cuinf_rope(_p(q), _p(k), _p(pos), S, nq, nk, theta, _stream()))


def kv_write_tail(k, v, ktail, vtail, slot, cnt):
    """Copy cnt tokens into the fp16 tail at slot  (kv_write_tail, engine.cu:190-198)."""
    nkv = ktail.shape[1]
    check(lib().cuinf_kv_write_tail(_p(k), _p(v), _p(ktail), _p(vtail), slot, cnt, nkv, _stream()))


def kv_commit_group(ktail, vtail, kc8, vc8, ksc, vsc, dst_tok_base, grp):
    """Commit a full 64-token tail to FP8 E4M3  (kv_commit_group, engine.cu:202-228)."""
    nkv = ktail.shape[1]
    check(lib().cuinf_kv_commit_group(_p(ktail), _p(vtail), _p(kc8), _p(vc8), _p(ksc), _p(vsc),
                                      dst_tok_base, grp, nkv, _stream()))


def attn_decode(q, kc8, vc8, ksc, vsc, ktail, vtail, committed, qpos, scale=0.125, out=None,
                workspace=None):
    """Flash-decoding attention of one token over FP8 groups + fp16 tail
    (attn_decode_split + attn_decode_combine, engine.cu:396-480).  q [nh,64]."""
    nh = q.numel() // 64
    nkv = ktail.shape[1]
    if out is None:
        out = torch.empty_like(q)
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(lib().cuinf_attn_decode(_p(q), _p(kc8), _p(vc8), _p(ksc), _p(vsc), _p(ktail), _p(vtail),
                                  committed, qpos, scale, _p(out), nh, nkv, _p(workspace), ws_bytes,
                                  _stream()))
    return out


def attn_decode_noalloc(q, kc8, vc8, ksc, vsc, ktail, vtail, committed, qpos, scale=0.125,
                        out=None):
    """attn_decode with the library's static 512 KiB scratch: the C call allocates
    no device memory (out is allocated here only when not given).  Calls on
    one device must not overlap."""
    nh = q.numel() // 64
    nkv = ktail.shape[1]
    if out is None:
        out = torch.empty_like(q)
    check(lib().cuinf_attn_decode_noalloc(_p(q), _p(kc8), _p(vc8), _p(ksc), _p(vsc), _p(ktail),
                                          _p(vtail), committed, qpos, scale, _p(out), nh, nkv,
                                          _stream()))
    return out


def conv_pre(inproj, C, Bx, S, H):
    """C = half(C), Bx = half(B*x) from in_proj rows B|C|x  (conv_pre, engine.cu:483-494)."""
    check(lib().cuinf_conv_pre(_p(inproj), _p(C), _p(Bx), S, H, _stream()))


def conv_apply(Bx, C, w, state, y, S, H):
    """Causal depthwise conv k=3 gated by C  (conv_apply, engine.cu:498-512)."""
    check(lib().cuinf_conv_apply(_p(Bx), _p(C), _p(w), _p(state), _p(y), S, H, _stream()))


def conv_update_state(Bx, state, S, H):
    """Keep the last two Bx  (conv_update_state, engine.cu:514-525)."""
    check(lib().cuinf_conv_update_state(_p(Bx), _p(state), S, H, _stream()))


def swiglu(g, u, out):
    """out = half(silu(g) * u)  (swiglu, engine.cu:542-547)."""
    check(lib().cuinf_swiglu(_p(g), _p(u), _p(out), g.numel(), _stream()))


def acc_scaled(dst, src, w):
    """dst = half(dst + w * src)  (acc_scaled, engine.cu:556-559)."""
    check(lib().cuinf_acc_scaled(_p(dst), _p(src), float(w), dst.numel(), _stream()))


def add_inplace(a, b):
    """a = half(a + b)  (add_inplace, engine.cu:527-530)."""
    check(lib().cuinf_add_inplace(_p(a), _p(b), a.numel(), _stream()))


def add_f32_inplace(a, b):
    """a = half(a + b_f32)  (add_f32_inplace, engine.cu:532-535)."""
    check(lib().cuinf_add_f32_inplace(_p(a), _p(b), a.numel(), _stream()))


def f32_to_f16(src, dst):
    """dst = half(src)  (f32_to_f16, engine.cu:537-540)."""
    check(lib().cuinf_f32_to_f16(_p(src), _p(dst), src.numel(), _stream()))


def embed_gather(embed, ids, out):
    """out[s,:] = embed[ids[s],:]  (embed_gather, engine.cu:549-554)."""
    H = embed.shape[1]
    check(lib().cuinf_embed_gather(_p(embed), _p(ids), _p(out), ids.numel(), H, _stream()))


def argmax(logits, out=None):
    """Index of the max logit with argmax_kernel's tie rule (engine.cu:562-572)."""
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=logits.device)
    check(lib().cuinf_argmax(_p(logits), logits.numel(), _p(out), _stream()))
    return out


def moe_route(logits, bias, topk, idx=None, w=None):
    """Sigmoid + expert bias, top-k, norm_topk_prob on the device
    (the host loop of engine.cu:883-892).  logits fp32 [S,E], bias fp16 [E]."""
    E = bias.numel()
    S = logits.numel() // E
    if idx is None:
        idx = torch.empty((S, topk), dtype=torch.int32, device=logits.device)
    if w is None:
        w = torch.empty((S, topk), dtype=torch.float32, device=logits.device)
    check(lib().cuinf_moe_route(_p(logits), _p(bias), S, E, topk, _p(idx), _p(w), _stream()))
    return idx, w


def expert_table(experts):
    """Device table of per-expert pointers for moe_ffn: experts is a list of
    (w1_packed, w1_scales, w3_packed, w3_scales, w2_packed, w2_scales)."""
    ptrs = [t.data_ptr() for e in experts for t in e]
    dev = experts[0][0].device
    return torch.tensor(ptrs, dtype=torch.int64, device=dev)


def moe_ffn(xn, gate, expert_bias, table, h, topk, moe_inter, idx=None, w=None):
    """Fused MoE FFN of one token, h updated in place (engine.cu:877-905)."""
    H = h.numel()
    E = expert_bias.numel()
    check(lib().cuinf_moe_ffn(_p(xn), _p(gate), _p(expert_bias), _p(table), _p(h), H, moe_inter, E,
                              topk, _p(idx), _p(w), None, 0, _stream()))


def quantize_int4(w):
    """INT4 G=128 export quantizer of tools/export_weights.py:64-79 on the device.

    w fp32 [N,K] CUDA -> (packed u8 [N,K/2], scales fp16 [N,K/128])."""
    _dt(w, torch.float32, "w")
    N, K = w.shape
    packed = torch.empty((N, K // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((N, K // 128), dtype=torch.float16, device=w.device)
    check(lib().cuinf_quantize_int4(_p(w), N, K, _p(packed), _p(scales), _stream()))
    return packed, scales


# --------------------------------------------------------------------------
# serving attention: packed prompts, and a paged FP8 cache
# --------------------------------------------------------------------------
# These checks run before kernels of a few microseconds, so each looks at a tensor's properties once.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _heads(t, name, index=None):
    """(pointer, elements between tokens, heads) of fp16 rows [T, heads, 64]; the
    tokens may be apart (a part of a wider row), a token's heads not."""
    if t.dtype is not torch.float16:
        raise TypeError(f"{name} must be {torch.float16}, got {t.dtype}")
    at = t.get_device()
    if at < 0:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if index is not None and at != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != 64 or shape[1] == 0:
        raise ValueError(f"{name} must be [tokens, heads, 64], got {tuple(shape)}")
    if stride[2] != 1 or (shape[1] > 1 and stride[1] != 64):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    return t.data_ptr(), stride[0] if shape[0] > 1 else shape[1] * 64, shape[1]


def _whole(t, dtype, shape, name, index):
    """Pointer of a contiguous tensor of this type and shape on this device."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")
    return t.data_ptr()


def _paged(index, n, table, kp8, vp8, kps, vps, ktail, vtail):
    """Checked pointers of a paged cache, in the order of the C ABI, and its sizes."""
    if table.dim() != 2 or table.shape[1] == 0:
        raise ValueError("table must be [sequences, pages]")
    pool = kp8.shape
    if len(pool) != 4 or pool[2] != 64 or pool[3] != 64 or pool[0] == 0 or pool[1] == 0:
        raise ValueError(f"kp8 must be [pages, kv heads, 64, 64], got {tuple(pool)}")
    n_pages, nkv = pool[0], pool[1]
    width = table.shape[1]
    u8, f16, tail = torch.uint8, torch.float16, (n, nkv, 64, 64)
    return (_whole(table, torch.int32, (n, width), "table", index), width,
            _whole(kp8, u8, pool, "kp8", index), _whole(vp8, u8, pool, "vp8", index),
            _whole(kps, f16, (n_pages, nkv), "kps", index), _whole(vps, f16, (n_pages, nkv), "vps", index), n_pages,
            _whole(ktail, f16, tail, "ktail", index), _whole(vtail, f16, tail, "vtail", index)), nkv


def _cu(cu_seqlens, index):
    shape = cu_seqlens.shape
    if len(shape) != 1 or shape[0] < 1:
        raise ValueError("cu_seqlens must be [sequences + 1]")
    return _whole(cu_seqlens, torch.int32, shape, "cu_seqlens", index), shape[0] - 1


def _out(out, q, index):
    if out is None:
        out = torch.empty_like(q)
    return out, _whole(out, torch.float16, q.shape, "out", index)


@functools.lru_cache(maxsize=256)
def _scratch_bytes(fn, *args):
    return getattr(lib(), fn)(*args)


def _scratch(workspace, size, like, index):
    """(workspace, its pointer and bytes); without one, scratch of this call (from
    torch's allocator, so it follows the stream's order and a capture's pool)."""
    if workspace is None:
        if size == 0:
            return None, None, 0
        workspace = like.new_empty(size, dtype=torch.uint8)
    elif workspace.get_device() != index or not workspace.is_contiguous():
        raise ValueError(f"workspace: expected a contiguous tensor on cuda:{index}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _call(fn, index, *args):
    """A C entry on the device `index` and torch's current stream there."""
    if torch.cuda.current_device() == index:
        check(fn(*args, _raw_stream(index)))
    else:
        with torch.cuda.device(index):
            check(fn(*args, _raw_stream(index)))


def attn_varlen(q, k, v, cu_seqlens, scale=0.125, out=None, workspace=None):
    """Causal attention of prompts packed behind one another: row t of sequence s
    (rows cu_seqlens[s]..cu_seqlens[s+1]-1) attends that sequence's rows up to t.

    q fp16 [T,nh,64], k, v fp16 [T,nkv,64] (tokens may be strided, so k and v may
    be parts of one projection's rows), cu_seqlens int32 [n+1] on the device;
    query head h reads kv head h // (nh // nkv).  Rows outside all sequences are
    left as they were (undefined in a new `out`).  Nothing synchronizes."""
    qp, qs, nh = _heads(q, "q")
    index = q.get_device()
    kp, ks, nkv = _heads(k, "k", index)
    vp, vs, nv = _heads(v, "v", index)
    T = q.shape[0]
    if k.shape[0] != T or v.shape[0] != T or nv != nkv:
        raise ValueError("q, k and v must have the same tokens, k and v the same heads")
    cu, n = _cu(cu_seqlens, index)
    out, op = _out(out, q, index)
    if T == 0 or n == 0:
        return out
    workspace, ws, nbytes = _scratch(workspace, _scratch_bytes("cuinf_attn_varlen_workspace_size", n, T, nh, nkv), q,
                                     index)
    _call(lib().cuinf_attn_varlen, index, qp, qs, kp, ks, vp, vs, cu, n, T, scale, op, nh, nkv, ws, nbytes)
    return out


def kv_paged_append(k, v, cu_seqlens, ctx_lens, table, kp8, vp8, kps, vps, ktail, vtail):
    """Append packed new rows to the paged FP8 cache, what kv_write_tail and
    kv_commit_group do for one sequence's contiguous cache.

    k, v fp16 [T,nkv,64] (tokens may be strided); sequence s holds ctx_lens[s]
    tokens before and gets rows cu_seqlens[s]..cu_seqlens[s+1]-1.  Groups of 64
    tokens that become complete are quantized into page table[s, group] (kp8/vp8
    u8 [pages,nkv,64,64], kps/vps fp16 [pages,nkv]); the rest goes to
    ktail/vtail fp16 [n,nkv,64,64].  Page indices outside the pool and lengths
    outside their ranges are skipped and reported by paged_error()."""
    kp, ks, nkv = _heads(k, "k")
    index = k.get_device()
    vp, vs, nv = _heads(v, "v", index)
    T = k.shape[0]
    if v.shape[0] != T or nv != nkv:
        raise ValueError("k and v must have the same shape")
    cu, n = _cu(cu_seqlens, index)
    ctx = _whole(ctx_lens, torch.int32, (n,), "ctx_lens", index)
    cache, cache_kv = _paged(index, n, table, kp8, vp8, kps, vps, ktail, vtail)
    if cache_kv != nkv:
        raise ValueError(f"the cache has {cache_kv} kv heads, k {nkv}")
    if T == 0 or n == 0:
        return
    _call(lib().cuinf_kv_paged_append, index, kp, ks, vp, vs, cu, ctx, n, T, *cache, nkv)


def attn_paged(q, cu_seqlens, kv_lens, table, kp8, vp8, kps, vps, ktail, vtail, scale=0.125, max_q=None, out=None,
               workspace=None):
    """Attention of new tokens over the paged FP8 cache that already holds them
    (kv_paged_append first): sequence s has kv_lens[s] tokens, its new rows
    q[cu_seqlens[s]:cu_seqlens[s+1]] are the last of them, and each attends all
    positions up to its own; a row whose position is negative is zero.

    q fp16 [T,nh,64] (tokens may be strided); a chunk of a prompt, drafted
    tokens, or one token per sequence (the decode step), mixed as they come.
    max_q: an upper bound of the rows of one sequence (default T); a smaller
    bound lets a pure decode step skip the chunks' kernel.  Nothing
    synchronizes; what the device finds wrong is reported by paged_error()."""
    qp, qs, nh = _heads(q, "q")
    index = q.get_device()
    cu, n = _cu(cu_seqlens, index)
    kvl = _whole(kv_lens, torch.int32, (n,), "kv_lens", index)
    cache, nkv = _paged(index, n, table, kp8, vp8, kps, vps, ktail, vtail)
    out, op = _out(out, q, index)
    T = q.shape[0]
    if T == 0 or n == 0:
        return out
    max_q = T if max_q is None else min(max_q, T)  # (a bound above 32 bits would wrap in the call)
    size = _scratch_bytes("cuinf_attn_paged_workspace_size", n, T, max_q, nh, nkv, cache[1])
    workspace, ws, nbytes = _scratch(workspace, size, q, index)
    _call(lib().cuinf_attn_paged, index, qp, qs, cu, kvl, n, T, max_q, *cache, scale, op, nh, nkv, ws, nbytes)
    return out


def paged_error():
    """Read and clear the current device's error word of attn_varlen,
    kv_paged_append and attn_paged (0 = none; the bits are in cuinf.h).  Waits
    for all work of the device, on every stream."""
    flags = ctypes.c_uint(0)
    check(lib().cuinf_paged_error(ctypes.byref(flags)))
    return flags.value
