"""Refusals of the serving attention operators (attn_varlen, kv_paged_append,
attn_paged) that need no GPU: the C entry points' argument checks with host
pointers that are never read, and the Python wrappers' checks of types, shapes
and devices."""
import ctypes

import pytest
import torch

from cuda_inf_b200 import _lib, ops

BUF = ctypes.create_string_buffer(64)
P = (ctypes.addressof(BUF) + 15) // 16 * 16


def varlen(q=P, qs=2048, k=P, ks=512, v=P, vs=512, cu=P, n=1, rows=4, scale=0.125, out=P, nh=32, nkv=8, ws=P,
           wb=1 << 40):
    L = _lib.lib()
    return L.cuinf_attn_varlen(q, qs, k, ks, v, vs, cu, n, rows, scale, out, nh, nkv, ws, wb, None), L.cuinf_last_error()


def append(k=P, ks=512, v=P, vs=512, cu=P, ctx=P, n=1, rows=4, table=P, width=4, kp8=P, vp8=P, kps=P, vps=P, pages=4,
           ktail=P, vtail=P, nkv=8):
    L = _lib.lib()
    return L.cuinf_kv_paged_append(k, ks, v, vs, cu, ctx, n, rows, table, width, kp8, vp8, kps, vps, pages, ktail,
                                   vtail, nkv, None), L.cuinf_last_error()


def paged(q=P, qs=2048, cu=P, kv=P, n=1, rows=4, max_q=4, table=P, width=4, kp8=P, vp8=P, kps=P, vps=P, pages=4,
          ktail=P, vtail=P, scale=0.125, out=P, nh=32, nkv=8, ws=P, wb=1 << 40):
    L = _lib.lib()
    return L.cuinf_attn_paged(q, qs, cu, kv, n, rows, max_q, table, width, kp8, vp8, kps, vps, pages, ktail, vtail,
                              scale, out, nh, nkv, ws, wb, None), L.cuinf_last_error()


HEADS = b"nh must be a multiple of nkv"
CASES = [
    (varlen, dict(q=None), b"null pointer"), (varlen, dict(cu=None), b"null pointer"),
    (varlen, dict(out=None), b"null pointer"), (varlen, dict(n=0), b"must be positive"),
    (varlen, dict(rows=0), b"must be positive"), (varlen, dict(rows=-3), b"must be positive"),
    (varlen, dict(scale=0.0), b"scale must be"), (varlen, dict(scale=-1.0), b"scale must be"),
    (varlen, dict(scale=float("nan")), b"scale must be"), (varlen, dict(scale=float("inf")), b"scale must be"),
    (varlen, dict(nh=30), HEADS), (varlen, dict(nkv=0), HEADS), (varlen, dict(nh=129, nkv=1, qs=8256), HEADS),
    (varlen, dict(q=P + 2), b"q: 16-byte aligned"), (varlen, dict(k=P + 8), b"k: 16-byte aligned"),
    (varlen, dict(qs=2040), b"q: 16-byte aligned"), (varlen, dict(ks=513), b"k: 16-byte aligned"),
    (varlen, dict(vs=64), b"v: 16-byte aligned"), (varlen, dict(out=P + 2), b"out must be 16-byte"),
    (append, dict(k=None), b"null pointer"), (append, dict(ctx=None), b"null pointer"),
    (append, dict(table=None), b"null pointer"), (append, dict(vps=None), b"null pointer"),
    (append, dict(n=-1), b"must be positive"), (append, dict(rows=0), b"must be positive"),
    (append, dict(pages=0), b"must be positive"), (append, dict(width=0), b"must be positive"),
    (append, dict(kp8=P + 4), b"pages and tails must be"), (append, dict(vtail=P + 8), b"pages and tails must be"),
    (append, dict(kps=P + 1), b"misaligned scales"), (append, dict(vs=8), b"v: 16-byte aligned"),
    (append, dict(nkv=0), HEADS),
    (append, dict(width=1 << 25), b"table_width"), (paged, dict(width=1 << 25), b"table_width"),
    (varlen, dict(rows=4096, wb=100), b"workspace"), (varlen, dict(rows=4096, ws=None), b"workspace"),
    (paged, dict(width=64, wb=100), b"workspace"), (paged, dict(width=64, ws=P + 4), b"workspace"),
    (paged, dict(kv=None), b"null pointer"), (paged, dict(ktail=None), b"null pointer"),
    (paged, dict(max_q=0), b"max_q must be"), (paged, dict(scale=float("inf")), b"scale must be"),
    (paged, dict(nh=12), HEADS), (paged, dict(out=P + 4), b"out must be 16-byte"),
    (paged, dict(qs=2041), b"q: 16-byte aligned"), (paged, dict(pages=-1), b"must be positive"),
]


@pytest.mark.parametrize("call,bad,msg", CASES, ids=[f"{c.__name__}-{next(iter(b))}-{i}" for i, (c, b, _) in
                                                     enumerate(CASES)])
def test_c_entry_refuses(call, bad, msg):
    rc, err = call(**bad)
    assert rc == 1 and msg in err, (rc, err)


def test_error_word_refuses_null():
    assert _lib.lib().cuinf_paged_error(None) == 1


def _t(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def test_wrappers_refuse_cpu_tensors_and_types():
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attn_varlen(_t(4, 4, 64), _t(4, 1, 64), _t(4, 1, 64), cu)
    with pytest.raises(TypeError, match="q must be"):
        ops.attn_varlen(_t(4, 4, 64).bfloat16(), _t(4, 1, 64), _t(4, 1, 64), cu)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_paged_append(_t(4, 1, 64), _t(4, 1, 64), cu, cu[:1], cu[None], *(None,) * 6)
    with pytest.raises(TypeError, match="q must be"):
        ops.attn_paged(_t(4, 4, 64).float(), cu, cu[:1], cu[None], *(None,) * 6)


@pytest.mark.parametrize("call", [varlen, paged])
@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scale_that_is_infinite_in_powers_of_two(call, scale):
    """Scores are taken times log2(e): a scale that this makes infinite would give no numbers."""
    rc, err = call(scale=scale)
    assert rc == 1 and b"scale must be" in err, (rc, err)
