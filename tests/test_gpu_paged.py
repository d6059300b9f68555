"""GPU tests of the serving attention operators against plain 64-bit forms.

Tolerance of the attention, per output value, from the formulas: the softmax
weights are rounded to fp16 before they meet the values, each off by at most
2^-11 of itself, so the sum is off by 2^-11 sum p|v|; their exponentials, the
scores' fp32 sums and the running rescalings are together well below another
2^-12 of each weight for scores up to 2^7; the result is rounded to fp16
(2^-11 |o|).  Weights below fp16's normal range are off by at most 2^-25 of the
largest weight each, in units of which the values enter with at most max|v|
(for FP8 pages the weight carries the page's scale times a constant of at least
16, so a value of at most 448 scales enters with 28).  Hence
  |got - o| <= 2^-11 |o| + 1.5 * 2^-11 sum p|v| + n 2^-25 max(max|v|, 28).
Codes, scales and tails of the cache have to be those of kv_commit_group and
kv_write_tail, bit for bit.
"""
import pytest
import torch

from cuda_inf_b200 import ops
from cuda_inf_b200._lib import CuinfError

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _clean(cuda):
    ops.paged_error()
    yield
    torch.cuda.synchronize()


# ------------------------------------------------------------------ plain forms
def plain_rows(q, k, v, first, scale):
    """q [c,nh,64] at positions first.., k, v [nkv,l,64] (64 bits): (out, bound on its error)."""
    c, nh, _ = q.shape
    k, v = (x.repeat_interleave(nh // k.shape[0], 0) for x in (k, v))
    s = torch.einsum("chd,hld->hcl", q.double(), k) * scale
    pos = first + torch.arange(c, device=q.device)
    ok = (torch.arange(k.shape[1], device=q.device)[None] <= pos[:, None])[None]
    s = torch.where(ok, s, torch.full_like(s, -INF))
    p = torch.where(pos[None, :, None] >= 0, torch.softmax(s, -1), torch.zeros_like(s)) if k.shape[1] else s
    # a weight of zero takes no part, whatever its value is
    fin = torch.isfinite(v)
    o = torch.einsum("hcl,hld->chd", p, torch.where(fin, v, torch.zeros_like(v)))
    mag = torch.einsum("hcl,hld->chd", p, torch.where(fin, v, torch.zeros_like(v)).abs())
    if not bool(fin.all()):
        seen = ok.double().expand_as(s)
        for kind, x in ((v == INF, INF), (v == -INF, -INF), (v.isnan(), NAN)):
            hit = torch.einsum("hcl,hld->chd", seen, kind.double()) > 0
            o = torch.where(hit, o + x, o)
    big = float(torch.where(fin, v, torch.zeros_like(v)).abs().max()) if v.numel() else 0.0
    return o, 2.0**-11 * o.abs() + 1.5 * 2.0**-11 * mag + k.shape[1] * 2.0**-25 * max(big, 28.0)


def close(got, want, tol):
    g = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    assert torch.equal(g[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    e = (g - want).abs()[fin]
    bad = e > tol[fin]
    assert not bool(bad.any()), (float(e.max()), float((e / tol[fin]).max()), int(bad.sum()), e.numel())


def cum(lens, dev, start=0):
    c = [start]
    for x in lens:
        c.append(c[-1] + x)
    return torch.tensor(c, dtype=torch.int32, device=dev)


def rnd(shape, seed, dev, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).half()


# ------------------------------------------------------------------ packed prompts
def check_varlen(q, k, v, lens, out, scale=0.125, start=0):
    a = start
    for x in lens:
        if x:
            o, tol = plain_rows(q[a:a + x], k[a:a + x].double().transpose(0, 1), v[a:a + x].double().transpose(0, 1), 0,
                                scale)
            close(out[a:a + x], o, tol)
        a += x


LENS = [[1], [2], [17], [64], [127], [128], [129], [255, 1, 0, 3], [300], [1, 1, 1, 1, 1], [513, 64, 31, 0, 0, 700],
        [1025, 130], [2500], [40] * 37, [0, 0, 5]]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:6])))
@pytest.mark.parametrize("nh,nkv", [(32, 8), (4, 1), (8, 8), (12, 4), (5, 1), (32, 1), (7, 7)])
def test_varlen(cuda, lens, nh, nkv):
    t = sum(lens)
    q, k, v = rnd((t, nh, 64), 1 + t, cuda), rnd((t, nkv, 64), 2 + t, cuda), rnd((t, nkv, 64), 3 + t, cuda)
    out = ops.attn_varlen(q, k, v, cum(lens, cuda))
    assert ops.paged_error() == 0
    check_varlen(q, k, v, lens, out)


@pytest.mark.parametrize("grp", [96, 128, 48])
def test_varlen_many_heads_per_kv_head(cuda, grp):
    lens = [130, 5]
    q, k, v = rnd((135, grp, 64), 1, cuda), rnd((135, 1, 64), 2, cuda), rnd((135, 1, 64), 3, cuda)
    check_varlen(q, k, v, lens, ops.attn_varlen(q, k, v, cum(lens, cuda)))


def test_varlen_strided_rows_and_out(cuda):
    """q, k and v as parts of wider rows, out given; rows outside the sequences stay."""
    lens, start, t = [70, 0, 200], 9, 300
    wide = rnd((t, 20, 64), 5, cuda)
    q, k, v = wide[:, :12], wide[:, 12:16], wide[:, 16:]
    out = torch.full((t, 12, 64), 7.0, dtype=torch.float16, device=cuda)
    assert ops.attn_varlen(q, k, v, cum(lens, cuda, start), out=out) is out
    check_varlen(q, k, v, lens, out, start=start)
    assert bool((out[:start] == 7).all()) and bool((out[start + 270:] == 7).all())


@pytest.mark.parametrize("scale,mul", [(0.125, 8.0), (1.0, 3.0), (1e-4, 1.0), (0.125, 0.0)])
def test_varlen_scores(cuda, scale, mul):
    """Scores that are sharp, flat, all equal; a maximum that grows along the keys."""
    lens = [400, 33]
    q, k, v = rnd((433, 8, 64), 1, cuda, mul), rnd((433, 2, 64), 2, cuda), rnd((433, 2, 64), 3, cuda)
    k = k * torch.linspace(0.1, 1.5, 433, device=cuda).half()[:, None, None]
    check_varlen(q, k, v, lens, ops.attn_varlen(q, k, v, cum(lens, cuda), scale=scale), scale=scale)


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("at", [0, 63, 64, 190, 299])
def test_varlen_masked_places_do_not_reach_the_rows(cuda, bad, at):
    """A value that is no number reaches the rows that attend it, and those alone;
    keys that are no numbers in masked places reach nothing."""
    lens, nh, nkv = [300, 45], 8, 2
    q, k, v = rnd((345, nh, 64), 1, cuda), rnd((345, nkv, 64), 2, cuda), rnd((345, nkv, 64), 3, cuda)
    v[at, 1, 5] = bad
    out = ops.attn_varlen(q, k, v, cum(lens, cuda))
    check_varlen(q, k, v, lens, out)
    k[at] = bad  # rows before `at` and the other sequence stay as they were
    out2 = ops.attn_varlen(q, k, v, cum(lens, cuda))
    assert torch.equal(out2[:at], out[:at]) and torch.equal(out2[300:], out[300:])
    assert bool(out2[at].isnan().all())


def test_varlen_neighbours_of_nan(cuda):
    """Sequences of NaN on both sides of one of numbers."""
    lens = [100, 77, 300]
    q, k, v = rnd((477, 8, 64), 1, cuda), rnd((477, 2, 64), 2, cuda), rnd((477, 2, 64), 3, cuda)
    want = ops.attn_varlen(q, k, v, cum(lens, cuda))
    for t in (q, k, v):
        t[:100] = NAN
        t[177:] = NAN
    out = ops.attn_varlen(q, k, v, cum(lens, cuda))
    assert torch.equal(out[100:177], want[100:177])
    assert bool(out[:100].isnan().all()) and bool(out[177:].isnan().all())


def test_varlen_bad_offsets_are_reported(cuda):
    q, k, v = rnd((50, 4, 64), 1, cuda), rnd((50, 1, 64), 2, cuda), rnd((50, 1, 64), 3, cuda)
    want = ops.attn_varlen(q, k, v, cum([50], cuda))
    assert ops.paged_error() == 0
    out = torch.full_like(want, 3.0)
    ops.attn_varlen(q, k, v, torch.tensor([0, 50, 70], dtype=torch.int32, device=cuda), out=out)
    assert ops.paged_error() & 4
    assert torch.equal(out, want)
    assert ops.paged_error() == 0


# ------------------------------------------------------------------ the paged cache
class Cache:
    """Pages in a shuffled order for n sequences of up to `room` tokens each."""

    def __init__(self, n, nkv, room, dev, seed=0, spare=2):
        w = max(1, -(-room // 64))
        g = torch.Generator(device=dev).manual_seed(seed)
        self.n, self.nkv, self.dev = n, nkv, dev
        pages = n * w + spare
        self.table = torch.randperm(pages, generator=g, device=dev)[:n * w].to(torch.int32).view(n, w).contiguous()
        # free places hold codes and bits that are no numbers
        self.kp8 = torch.full((pages, nkv, 64, 64), 0x7F, dtype=torch.uint8, device=dev)
        self.vp8 = self.kp8.clone()
        self.kps = torch.full((pages, nkv), NAN, dtype=torch.float16, device=dev)
        self.vps = self.kps.clone()
        self.ktail = torch.full((n, nkv, 64, 64), NAN, dtype=torch.float16, device=dev)
        self.vtail = self.ktail.clone()
        self.lens = [0] * n

    @property
    def t(self):
        return self.table, self.kp8, self.vp8, self.kps, self.vps, self.ktail, self.vtail

    def ints(self):
        return torch.tensor(self.lens, dtype=torch.int32, device=self.dev)

    def append(self, k, v, new):
        ops.kv_paged_append(k, v, cum(new, self.dev), self.ints(), *self.t)
        self.lens = [a + b for a, b in zip(self.lens, new)]

    def values(self, i, which):
        """[nkv, len, 64] in 64 bits."""
        g, r = divmod(self.lens[i], 64)
        p8, ps, tail = (self.kp8, self.kps, self.ktail) if which == "k" else (self.vp8, self.vps, self.vtail)
        at = self.table[i, :g].long()
        x = p8[at].view(torch.float8_e4m3fn).double() * ps[at].double()[:, :, None, None]
        x = x.permute(1, 0, 2, 3).reshape(self.nkv, g * 64, 64)
        return torch.cat([x, tail[i, :, :r].double()], 1)

    def check(self, q, new, out, scale=0.125):
        a = 0
        for i, c in enumerate(new):
            if c:
                o, tol = plain_rows(q[a:a + c], self.values(i, "k"), self.values(i, "v"), self.lens[i] - c, scale)
                close(out[a:a + c], o, tol)
            a += c

    def attend(self, q, new, **kw):
        return ops.attn_paged(q, cum(new, self.dev), self.ints(), *self.t, **kw)


def fill(cache, lens, seed, vscale=0.5):
    """Appends `lens` random tokens in one call."""
    t = sum(lens)
    if t:
        cache.append(rnd((t, cache.nkv, 64), seed, cache.dev), rnd((t, cache.nkv, 64), seed + 1, cache.dev, vscale),
                     lens)


APPENDS = [([0], [1]), ([0], [64]), ([0], [63]), ([63], [1]), ([63], [2]), ([5], [59]), ([5], [60]), ([0], [65]),
           ([60], [200]), ([10, 0, 64, 127], [1, 1, 1, 1]), ([10, 0, 64, 127, 3], [300, 0, 64, 129, 0]),
           ([1] * 300, [1] * 300), ([0, 7], [1500, 1])]


@pytest.mark.parametrize("ctx,new", APPENDS, ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("nkv", [1, 8])
def test_append_is_write_tail_and_commit(cuda, ctx, new, nkv):
    """Bit-equal to kv_write_tail + kv_commit_group, one sequence after another."""
    n = len(ctx)
    c = Cache(n, nkv, max(a + b for a, b in zip(ctx, new)) + 1, cuda, seed=len(ctx))
    fill(c, ctx, 11)
    kt, vt = c.ktail.clone(), c.vtail.clone()
    p = [x.clone() for x in (c.kp8, c.vp8, c.kps, c.vps)]
    wide = rnd((sum(new), 2 * nkv, 64), 21, cuda)
    k, v = wide[:, :nkv], wide[:, nkv:]
    old = list(c.lens)
    c.append(k, v, new)
    assert ops.paged_error() == 0
    at = 0
    for i in range(n):
        t1, t2 = (x[i].transpose(0, 1).clone(memory_format=torch.contiguous_format) for x in (kt, vt))  # [64, nkv, 64]
        done = 0
        while done < new[i]:
            pos = old[i] + done
            slot, cnt = pos % 64, min(64 - pos % 64, new[i] - done)
            ops.kv_write_tail(k[at + done:at + done + cnt].contiguous(), v[at + done:at + done + cnt].contiguous(),
                              t1, t2, slot, cnt)
            done += cnt
            if slot + cnt == 64:
                k8, v8 = (torch.empty((64, nkv, 64), dtype=torch.uint8, device=cuda) for _ in range(2))
                s1, s2 = (torch.empty((1, nkv), dtype=torch.float16, device=cuda) for _ in range(2))
                ops.kv_commit_group(t1, t2, k8, v8, s1, s2, 0, 0)
                page = int(c.table[i, pos // 64])
                p[0][page], p[1][page] = k8.transpose(0, 1), v8.transpose(0, 1)
                p[2][page], p[3][page] = s1[0], s2[0]
        rest = (old[i] + new[i]) % 64 if (old[i] + new[i]) // 64 > old[i] // 64 else old[i] % 64 + new[i]
        kt[i, :, :rest], vt[i, :, :rest] = t1.transpose(0, 1)[:, :rest], t2.transpose(0, 1)[:, :rest]
        at += new[i]
    for got, want in zip((c.kp8, c.vp8, c.kps, c.vps, c.ktail, c.vtail), (*p, kt, vt)):
        assert torch.equal(got.view(torch.uint8) if got.dtype != torch.uint8 else got,
                           want.view(torch.uint8) if want.dtype != torch.uint8 else want)


def test_append_zero_and_extreme_rows(cuda):
    """A page of zeros, of fp16's largest values, of its smallest: codes and scales in 64 bits."""
    c = Cache(1, 4, 64, cuda)
    k = torch.zeros((64, 4, 64), dtype=torch.float16, device=cuda)
    k[:, 1] = 65504.0
    k[:, 2] = 6e-8
    k[3, 3, 9] = -2.0
    c.append(k, k, [64])
    s = k.double().abs().amax((0, 2)) / 448 + 1e-12
    page = int(c.table[0, 0])
    assert torch.allclose(c.kps[page].double(), s, rtol=2**-10, atol=2**-25)
    codes = c.kp8[page].view(torch.float8_e4m3fn).double()
    want = (k.double() / s[None, :, None]).transpose(0, 1)
    assert bool(((codes - want).abs() <= want.abs() * 2**-4 + 2**-10).all())
    assert torch.equal(c.kp8[page], c.vp8[page])


def test_append_infinities_and_nan_as_the_commit(cuda):
    """Pages with an infinite value, a NaN, both: codes and scales of kv_commit_group, bit for bit."""
    c = Cache(1, 4, 64, cuda)
    k = rnd((64, 4, 64), 3, cuda)
    k[5, 0, 7], k[6, 1, 8], k[7, 2, 9], k[8, 2, 3] = INF, NAN, -INF, NAN
    c.append(k, k.flip(1).contiguous(), [64])
    k8, v8 = (torch.empty((64, 4, 64), dtype=torch.uint8, device=cuda) for _ in range(2))
    ks, vs = (torch.empty((1, 4), dtype=torch.float16, device=cuda) for _ in range(2))
    ops.kv_commit_group(k, k.flip(1).contiguous(), k8, v8, ks, vs, 0, 0)
    page = int(c.table[0, 0])
    assert torch.equal(c.kp8[page], k8.transpose(0, 1)) and torch.equal(c.vp8[page], v8.transpose(0, 1))
    assert torch.equal(c.kps[page].view(torch.int16), ks[0].view(torch.int16))
    assert torch.equal(c.vps[page].view(torch.int16), vs[0].view(torch.int16))


def test_append_bad_page_and_lengths_are_reported(cuda):
    c = Cache(3, 2, 128, cuda)
    fill(c, [60, 60, 60], 5)
    c.table[1, 0] = -1
    before = c.kp8.clone()
    c.append(rnd((15, 2, 64), 1, cuda), rnd((15, 2, 64), 2, cuda), [5, 5, 5])
    assert ops.paged_error() == 2
    changed = (c.kp8 != before).flatten(1).any(1)
    assert sorted(changed.nonzero().flatten().tolist()) == sorted([int(c.table[0, 0]), int(c.table[2, 0])])
    # a group past the table's width, a negative length
    c = Cache(1, 2, 64, cuda)
    fill(c, [60], 5)
    c.append(rnd((100, 2, 64), 1, cuda), rnd((100, 2, 64), 2, cuda), [100])
    assert ops.paged_error() == 2
    c = Cache(1, 2, 64, cuda)
    c.lens = [-4]
    before = [x.clone() for x in c.t]
    c.append(rnd((100, 2, 64), 1, cuda), rnd((100, 2, 64), 2, cuda), [100])
    assert ops.paged_error() == 4
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, c.t))


TOKENS = [[1], [2], [63], [64], [65], [128], [129], [1000], [1, 64, 700, 3, 128], [4097, 5], [513] * 40, [9000],
          list(range(1, 150))]


@pytest.mark.parametrize("lens", TOKENS, ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("nh,nkv", [(32, 8), (4, 1), (8, 8), (12, 4), (10, 2), (16, 1), (32, 1)])
def test_single_tokens(cuda, lens, nh, nkv):
    c = Cache(len(lens), nkv, max(lens), cuda, seed=1)
    fill(c, lens, 3)
    new = [1] * len(lens)
    q = rnd((len(lens), nh, 64), 7, cuda)
    out = c.attend(q, new, max_q=1)
    assert ops.paged_error() == 0
    c.check(q, new, out)
    # the bound of the longest chunk changes the way, not the result's meaning
    c.check(q, new, c.attend(q, new))


CHUNKS = [([0], [1]), ([0], [64]), ([0], [300]), ([1], [2]), ([63], [2]), ([100], [28]), ([64], [64]), ([500], [33]),
          ([130, 0, 64, 1000, 7], [5, 129, 0, 1, 300]), ([2000, 2000], [700, 1]), ([4000], [257]),
          ([30] * 20, [3] * 20), ([1200] * 9, [1] * 8 + [400]), ([0], [1100])]


@pytest.mark.parametrize("ctx,new", CHUNKS, ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("nh,nkv", [(32, 8), (4, 1), (8, 8), (12, 4), (10, 2), (32, 1)])
def test_chunks(cuda, ctx, new, nh, nkv):
    c = Cache(len(ctx), nkv, max(a + b for a, b in zip(ctx, new)), cuda, seed=2)
    fill(c, ctx, 3)
    fill(c, new, 5)
    wide = rnd((sum(new), nh + 2, 64), 7, cuda)
    q = wide[:, 1:nh + 1]
    out = c.attend(q, new, max_q=max(new))
    assert ops.paged_error() == 0
    c.check(q, new, out)


def test_rows_before_the_first_key_are_zero(cuda):
    """More new rows than the cache holds: the first ones have no key at all."""
    c = Cache(3, 2, 128, cuda)
    fill(c, [40, 3, 0], 3)
    new = [100, 5, 2]
    q = rnd((107, 8, 64), 7, cuda)
    out = c.attend(q, new)
    assert ops.paged_error() == 0
    assert bool((out[:60] == 0).all()) and bool((out[100:102] == 0).all()) and bool((out[105:] == 0).all())
    c.check(q, new, out)


def test_rows_outside_the_sequences_stay(cuda):
    c = Cache(2, 2, 256, cuda)
    fill(c, [200, 90], 3)
    q = rnd((300, 8, 64), 7, cuda)
    for new in ([1, 1], [150, 3]):
        out = torch.full_like(q, 7.0)
        ops.attn_paged(q, cum(new, cuda, 20), c.ints(), *c.t, out=out, max_q=max(new))
        a, b = 20, 20 + sum(new)
        c.check(q[a:b], new, out[a:b])
        assert bool((out[:a] == 7).all()) and bool((out[b:] == 7).all())


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("chunk", [1, 40, 200])
def test_paged_masked_places(cuda, bad, chunk):
    """Junk behind the last token, and a later token of the chunk that is no number."""
    total = 333
    c = Cache(1, 2, 448, cuda)
    fill(c, [total], 3)
    c.vtail[:, :, total % 64:] = bad
    c.ktail[:, :, total % 64:] = bad
    q = rnd((chunk, 8, 64), 7, cuda)
    out = c.attend(q, [chunk])
    c.check(q, [chunk], out)
    if chunk > 1:
        c.vtail[0, :, total % 64 - 1, 3] = bad  # the newest token: the last row alone attends it
        got = c.attend(q, [chunk])
        assert torch.equal(got[:-1], out[:-1])
        c.check(q, [chunk], got)


def test_paged_bad_pages_count_as_absent(cuda):
    """A page index outside the pool: its keys are left out, and reported."""
    for chunk in (1, 60):
        c = Cache(2, 2, 512, cuda)
        fill(c, [500, 300], 3)
        q = rnd((2 * chunk, 8, 64), 7, cuda)
        want = c.attend(q, [chunk, chunk])
        for wrong in (-1, c.kp8.shape[0], 2**31 - 1, -2**31):
            keep = int(c.table[0, 2])
            c.table[0, 2] = wrong
            out = c.attend(q, [chunk, chunk], max_q=chunk)
            assert ops.paged_error() == 2
            assert torch.equal(out[chunk:], want[chunk:])
            c.table[0, 2] = keep
            k, v = (torch.cat([c.values(0, x)[:, :128], c.values(0, x)[:, 192:]], 1) for x in ("k", "v"))
            o, tol = plain_rows(q[:chunk], k, v, 500 - 64 - chunk, 0.125)
            close(out[:chunk], o, tol)


def test_paged_bad_lengths_are_reported(cuda):
    c = Cache(3, 2, 128, cuda)
    fill(c, [100, 100, 100], 3)
    q = rnd((3, 8, 64), 7, cuda)
    want = c.attend(q, [1, 1, 1])
    for wrong in (-1, 192, 10000, 2**31 - 1, -2**31):
        c.lens[1] = wrong
        for mq in (1, 64):
            out = torch.full_like(want, 5.0)
            c.attend(q, [1, 1, 1], max_q=mq, out=out)
            assert ops.paged_error() == 4
            assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and bool((out[1] == 5).all())
    c.lens[1] = 100
    out = torch.full((61, 8, 64), 5.0, dtype=torch.float16, device=cuda)
    q = rnd((61, 8, 64), 7, cuda)
    c.attend(q, [1, 59, 1], max_q=1, out=out)  # a longer sequence than the caller's bound
    assert ops.paged_error() == 4
    assert bool((out[1:60] == 5).all()) and not bool((out[0] == 5).any()) and not bool((out[60] == 5).any())


def test_pages_of_zeros_and_infinite_scales(cuda):
    """A page whose scale is 0 beside masked places, and pages with an infinite key or value (their scale is
    infinite): rows that do not attend them stay as they are."""
    for chunk in (1, 3, 200):
        c = Cache(1, 2, 448, cuda)
        k, v = rnd((300, 2, 64), 3, cuda), rnd((300, 2, 64), 4, cuda)
        k[64:128] = 0
        v[192:256] = 0
        c.append(k, v, [300])
        q = rnd((chunk, 8, 64), 7, cuda)
        out = c.attend(q, [chunk], max_q=chunk)
        c.check(q, [chunk], out)
        o, tol = plain_rows(q, c.values(0, "k"), c.values(0, "v"), 300 - chunk, 0.125)
        for x in (k, v):
            x[200, 1, 5] = INF
            c.lens = [0]
            c.append(k, v, [300])
            got = c.attend(q, [chunk], max_q=chunk)
            first = max(0, min(chunk, 192 - (300 - chunk)))  # rows before the page
            # the heads of the other kv head, and (to the bit where the values' scale, which the limit of the weights
            # goes by, is the same) the rows before the page
            assert torch.equal(got[:, :4], out[:, :4])
            assert x is v or torch.equal(got[:first], out[:first])
            close(got[:first], o[:first], tol[:first])
            assert bool(got[first:, 4:].isnan().any(-1).all())
            x[200, 1, 5] = 1.0
            c.lens = [0]


def test_large_values(cuda):
    """Values up to fp16's largest: the weights carry the scale."""
    c = Cache(2, 2, 448, cuda)
    k, v = rnd((700, 2, 64), 3, cuda, 3.0), rnd((700, 2, 64), 4, cuda, 1.0).clamp(-3, 3) * 21000
    k = k * torch.linspace(0.2, 1.5, 700, device=cuda).half()[:, None, None]
    c.append(k, v, [350, 350])
    for new in ([1, 1], [300, 290]):
        q = rnd((sum(new), 8, 64), 7, cuda)
        out = c.attend(q, new, max_q=max(new))
        assert bool(out.isfinite().all())
        c.check(q, new, out)


def test_many_sequences(cuda):
    """More sequences than a CTA has threads: their line is walked in two passes."""
    lens = [(37 * i) % 90 for i in range(1300)]
    t = sum(lens)
    q, k, v = rnd((t, 4, 64), 1, cuda), rnd((t, 1, 64), 2, cuda), rnd((t, 1, 64), 3, cuda)
    check_varlen(q, k, v, lens, ops.attn_varlen(q, k, v, cum(lens, cuda)))
    c = Cache(1300, 1, 128, cuda)
    c.append(k, v, lens)
    new = [min(x, 1 + 39 * (i % 7 == 0)) for i, x in enumerate(lens)]
    q = rnd((sum(new), 4, 64), 7, cuda)
    c.check(q, new, c.attend(q, new, max_q=max(new)))
    assert ops.paged_error() == 0


@pytest.mark.parametrize("nh,nkv,new", [(1, 1, 1), (2, 1, 1), (3, 1, 1), (5, 1, 1), (4, 1, 2), (4, 1, 4), (8, 8, 9)])
def test_long_context_joined_from_many_parts(cuda, nh, nkv, new):
    """One sequence over all SMs: 1 to 16 rows, whose parts 1 to 16 threads share."""
    c = Cache(1, nkv, 20000, cuda)
    fill(c, [19990], 3)
    q = rnd((new, nh, 64), 7, cuda, 2.0)
    out = c.attend(q, [new], max_q=new)
    c.check(q, [new], out)
    assert torch.equal(out, c.attend(q, [new], max_q=new))


@pytest.mark.parametrize("lens,new", [
    ([6000] + [300] * 5, [1] + [200] * 5),
    ([3000] * 40 + [70], [1] * 40 + [17]),
    ([64, 5000], [1, 900]),
    ([63, 130, 200, 255], [1, 130, 3, 60]),
    ([1, 4000, 1], [1, 1, 1]),
    ([2000, 0, 1500], [700, 0, 1500]),
])
def test_chunks_beside_single_tokens(cuda, lens, new):
    """Both kernels at once, each on its part of the SMs, whatever the work's ratio."""
    c = Cache(len(lens), 2, max(lens), cuda)
    fill(c, lens, 5)
    q = rnd((sum(new), 8, 64), 7, cuda)
    out = c.attend(q, new)
    c.check(q, new, out)
    for _ in range(3):
        assert torch.equal(out, c.attend(q, new))
    assert ops.paged_error() == 0


def test_workspace_contents_do_not_matter(cuda):
    c = Cache(3, 2, 4096, cuda)
    fill(c, [4000, 700, 65], 3)
    q, k, v = rnd((2000, 8, 64), 1, cuda), rnd((2000, 2, 64), 2, cuda), rnd((2000, 2, 64), 3, cuda)
    ws = torch.empty(40 << 20, dtype=torch.uint8, device=cuda)
    want = None
    for byte in (0, 255, 1):
        ws.fill_(byte)
        got = (c.attend(q[:3], [1, 1, 1], max_q=1, workspace=ws), c.attend(q[:500], [400, 90, 10], workspace=ws),
               ops.attn_varlen(q, k, v, cum([1500, 500], cuda), workspace=ws))
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(CuinfError, match="workspace"):
        ops.attn_varlen(q, k, v, cum([1500, 500], cuda), workspace=ws[:1000])


def test_shared_prefix_pages(cuda):
    c = Cache(2, 2, 640, cuda)
    fill(c, [512, 512], 3)
    c.table[1, :8] = c.table[0, :8]
    fill(c, [30, 77], 9)
    for new in ([1, 1], [30, 77]):
        q = rnd((sum(new), 8, 64), 7, cuda)
        c.check(q, new, c.attend(q, new, max_q=max(new)))


def test_prefill_then_decode_as_served(cuda):
    """Packed prompts through attn_varlen and into the cache, the rest of one prompt in chunks, then steps of
    one token beside it; every output in 64 bits from what the cache holds."""
    n, nh, nkv = 4, 32, 8
    c = Cache(n, nkv, 700, cuda)
    steps = [[130, 64, 1, 0], [1, 1, 1, 250], [1, 1, 1, 250], [1, 1, 1, 37], [1, 1, 1, 1], [1, 0, 1, 1]]
    for i, new in enumerate(steps):
        t = sum(new)
        q, k, v = rnd((t, nh, 64), i, cuda), rnd((t, nkv, 64), 50 + i, cuda), rnd((t, nkv, 64), 90 + i, cuda)
        if i == 0:
            check_varlen(q, k, v, new, ops.attn_varlen(q, k, v, cum(new, cuda)))
        c.append(k, v, new)
        c.check(q, new, c.attend(q, new, max_q=max(new)))
    assert ops.paged_error() == 0


@pytest.mark.parametrize("total", [1, 63, 200, 4095])
def test_matches_the_contiguous_operator(cuda, total):
    """attn_decode on the same cache laid out contiguously."""
    c = Cache(1, 8, total, cuda)
    fill(c, [total], 3)
    g = total // 64
    at = c.table[0, :max(g, 1)].long()
    k8, v8 = (x[at].transpose(1, 2).reshape(-1, 8, 64).contiguous() for x in (c.kp8, c.vp8))
    ks, vs = (x[at].contiguous() for x in (c.kps, c.vps))
    q = rnd((1, 32, 64), 7, cuda)
    kt, vt = (x[0].transpose(0, 1).contiguous().nan_to_num(0.0) for x in (c.ktail, c.vtail))
    want = ops.attn_decode(q[0], k8, v8, ks, vs, kt, vt, g * 64, total - 1)
    got = c.attend(q, [1], max_q=1)[0]
    o, tol = plain_rows(q, c.values(0, "k"), c.values(0, "v"), total - 1, 0.125)
    close(got, o[0], tol[0])
    assert float((got.float() - want.float()).abs().max()) <= 2e-3 * float(want.float().abs().max()) + float(tol.max())


def test_offsets_past_32_bits(cuda):
    """Pages whose bytes lie behind 2^32."""
    nkv, pages = 8, 131072 + 40
    c = Cache(1, nkv, 64 * 9, cuda)
    for name in ("kp8", "vp8"):
        setattr(c, name, torch.zeros((pages, nkv, 64, 64), dtype=torch.uint8, device=cuda))
    for name in ("kps", "vps"):
        setattr(c, name, torch.zeros((pages, nkv), dtype=torch.float16, device=cuda))
    c.table = (pages - 1 - 2 * torch.arange(9, device=cuda, dtype=torch.int32))[None].contiguous()
    fill(c, [530], 3)
    assert int(c.kp8[:131000].count_nonzero()) == 0
    for new in ([1], [70], [520]):
        q = rnd((new[0], 32, 64), 7, cuda)
        c.check(q, new, c.attend(q, new, max_q=new[0]))
    assert ops.paged_error() == 0


def test_rows_past_32_bits(cuda):
    """q and out of more than 2^31 elements, k and v strided past 2^31."""
    nh, nkv, t = 128, 1, 270000
    lens = [t - 300, 300]
    q = torch.zeros((t, nh, 64), dtype=torch.float16, device=cuda)
    wide = torch.zeros((t, 8192), dtype=torch.float16, device=cuda)
    k, v = wide[:, None, :64], wide[:, None, 64:128]
    q[-300:] = rnd((300, nh, 64), 1, cuda)
    wide[-300:, :128] = rnd((300, 128), 2, cuda)
    out = torch.zeros_like(q)
    # the long sequence is cut short: its rows before the last 100 are nobody's
    cu = torch.tensor([t - 400, t - 300, t], dtype=torch.int32, device=cuda)
    ops.attn_varlen(q, k, v, cu, out=out)
    check_varlen(q[-300:], k[-300:], v[-300:], [300], out[-300:])
    assert ops.paged_error() == 0


def test_same_bits_twice(cuda):
    c = Cache(9, 8, 5000, cuda)
    fill(c, [5000, 1, 70, 900, 64, 3000, 2, 700, 128], 3)
    for new in ([1] * 9, [300, 1, 5, 64, 1, 1, 1, 130, 1]):
        q = rnd((sum(new), 32, 64), 7, cuda)
        a = c.attend(q, new, max_q=max(new))
        for _ in range(3):
            assert torch.equal(a, c.attend(q, new, max_q=max(new)))
    q, k, v = rnd((3000, 32, 64), 1, cuda), rnd((3000, 8, 64), 2, cuda), rnd((3000, 8, 64), 3, cuda)
    a = ops.attn_varlen(q, k, v, cum([2000, 1000], cuda))
    assert torch.equal(a, ops.attn_varlen(q, k, v, cum([2000, 1000], cuda)))


def test_captured_step_follows_the_lengths(cuda):
    """A step captured once (append, attention; all lengths on the device) and replayed as the sequences grow, a
    second graph beside it on another stream."""
    n, nh, nkv = 6, 32, 8
    sides = []
    for side in range(2):
        c = Cache(n, nkv, 700, cuda, seed=side)
        fill(c, [60 + 3 * i + 200 * side for i in range(n)], 3 + side)
        st = torch.cuda.Stream()
        ctx, kvl, cu = c.ints(), c.ints(), cum([1] * n, cuda)
        q, k, v = (torch.zeros((n, h, 64), dtype=torch.float16, device=cuda) for h in (nh, nkv, nkv))
        st.wait_stream(torch.cuda.current_stream())

        def step(c=c, ctx=ctx, kvl=kvl, cu=cu, q=q, k=k, v=v):
            ops.kv_paged_append(k, v, cu, ctx, *c.t)
            ctx.add_(1)
            kvl.copy_(ctx)
            return ops.attn_paged(q, cu, kvl, *c.t, max_q=1)

        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = step()
        sides.append((c, st, g, q, k, v, out, step))  # step holds the lengths' tensors
    for i in range(8):
        for j, (c, st, g, q, k, v, out, _) in enumerate(sides):
            q.copy_(rnd(q.shape, 10 * i + j, cuda)), k.copy_(rnd(k.shape, 11 * i + j, cuda))
            v.copy_(rnd(v.shape, 12 * i + j, cuda))
        torch.cuda.synchronize()
        for c, st, g, *_ in sides:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for c, st, g, q, k, v, out, _ in sides:
            c.lens = [x + 1 for x in c.lens]
            c.check(q, [1] * n, out)
    assert ops.paged_error() == 0


def test_two_streams_at_once(cuda):
    c = Cache(3, 8, 4000, cuda)
    fill(c, [4000, 100, 2000], 3)
    q1, q2 = rnd((3, 32, 64), 7, cuda), rnd((600, 32, 64), 8, cuda)
    new2 = [300, 50, 250]
    w1, w2 = c.attend(q1, [1] * 3, max_q=1), c.attend(q2, new2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    cu1, cu2, kvl = cum([1] * 3, cuda), cum(new2, cuda), c.ints()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            a = ops.attn_paged(q1, cu1, kvl, *c.t, max_q=1)
        with torch.cuda.stream(s2):
            b = ops.attn_paged(q2, cu2, kvl, *c.t)
        torch.cuda.synchronize()
        assert torch.equal(a, w1) and torch.equal(b, w2)


def test_empty_calls(cuda):
    q, k = rnd((0, 8, 64), 1, cuda), rnd((0, 2, 64), 1, cuda)
    assert ops.attn_varlen(q, k, k, cum([], cuda)).shape == (0, 8, 64)
    assert ops.attn_varlen(q, k, k, cum([0, 0], cuda)).shape == (0, 8, 64)
    c = Cache(2, 2, 64, cuda)
    c.append(k, k, [0, 0])
    assert c.attend(q, [0, 0]).shape == (0, 8, 64)
    q, k = rnd((5, 8, 64), 1, cuda), rnd((5, 2, 64), 1, cuda)
    out = torch.full_like(q, 2.0)
    ops.attn_varlen(q, k, k, cum([0, 0, 0], cuda), out=out)
    assert bool((out == 2).all()) and ops.paged_error() == 0


def test_refusals(cuda):
    c = Cache(2, 2, 64, cuda)
    q, k, cu = rnd((2, 8, 64), 1, cuda), rnd((2, 2, 64), 1, cuda), cum([1, 1], cuda)
    kvl = torch.ones(2, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="same tokens"):
        ops.attn_varlen(q, k[:1], k[:1], cu)
    with pytest.raises(CuinfError, match="multiple of nkv"):
        ops.attn_varlen(q[:, :7], k, k, cu)
    with pytest.raises(ValueError, match="heads must be contiguous"):
        ops.attn_varlen(q[:, ::2], k, k, cu)
    with pytest.raises(ValueError, match="64"):
        ops.attn_varlen(q[..., :32], k, k, cu)
    with pytest.raises(TypeError, match="cu_seqlens"):
        ops.attn_varlen(q, k, k, cu.long())
    with pytest.raises(CuinfError, match="16-byte aligned"):
        wide = rnd((2, 8 * 64 + 4), 1, cuda)
        ops.attn_varlen(wide[:, :512].view(2, 8, 64), k, k, cu)
    with pytest.raises(ValueError, match="out must be"):
        ops.attn_varlen(q, k, k, cu, out=q[:1].contiguous())
    with pytest.raises(CuinfError, match="scale"):
        ops.attn_varlen(q, k, k, cu, scale=0.0)
    with pytest.raises(ValueError, match="kv heads"):
        ops.kv_paged_append(k[:, :1], k[:, :1], cu, kvl, *c.t)
    with pytest.raises(ValueError, match="ctx_lens"):
        ops.kv_paged_append(k, k, cu, kvl[:1], *c.t)
    with pytest.raises(ValueError, match="table"):
        ops.attn_paged(q, cu, kvl, c.table[:1], *c.t[1:])
    with pytest.raises(TypeError, match="kp8"):
        ops.attn_paged(q, cu, kvl, c.table, c.kp8.half(), *c.t[2:])
    with pytest.raises(ValueError, match="vtail"):
        ops.attn_paged(q, cu, kvl, *c.t[:6], c.vtail[:1])
    with pytest.raises(CuinfError, match="max_q"):
        ops.attn_paged(q, cu, kvl, *c.t, max_q=0)


# ------------------------------------------------------------------ values of every size
def plain_weights(q, k, v, first, scale=0.125):
    """q [c,nh,64] at positions first.., k, v [nkv,l,64] (64 bits, finite): (out, bound on its error).

    The bound in units of each row's own weights w (they sum to 1) and values: a weight is rounded once to 11 bits
    (2^-11 of itself; its exponential, the scores' sums and the rescalings together stay below half of that), the
    result to fp16 (2^-11 |o|, or 2^-25 below its normal range), and what a weight loses below fp16's range is at
    most 2^-31 of the row's largest weight (2^-25 for the up to 63 keys of the tail) times its largest value."""
    c, nh, _ = q.shape
    k, v = (x.repeat_interleave(nh // k.shape[0], 0) for x in (k, v))
    s = torch.einsum("chd,hld->hcl", q.double(), k) * scale
    pos = first + torch.arange(c, device=q.device)
    ok = (torch.arange(k.shape[1], device=q.device)[None] <= pos[:, None])[None]
    w = torch.softmax(torch.where(ok, s, torch.full_like(s, -INF)), -1)
    o, mag = torch.einsum("hcl,hld->chd", w, v), torch.einsum("hcl,hld->chd", w, v.abs())
    top = (w.amax(-1) * v.abs().amax(-1).cummax(-1).values[:, pos]).T[..., None]
    lost = (k.shape[1] * 2.0**-31 + 63 * 2.0**-25) * top
    return o, 2.0**-11 * o.abs() + 1.5 * 2.0**-11 * mag + lost + 2.0**-25


def check_weights(c, q, new, out):
    a = 0
    for i, x in enumerate(new):
        if x:
            close(out[a:a + x], *plain_weights(q[a:a + x], c.values(i, "k"), c.values(i, "v"), c.lens[i] - x))
        a += x


def first_key_heavy(c, lens, sizes, weight, seed):
    """Fills the cache: keys of unit scores but for the first, which takes all but about n e^0.5 / e^weight of a
    row's weight and whose value is small beside the others, and values of standard deviation sizes[i] in the i-th
    equal part of a sequence."""
    for i, n in enumerate(lens):
        k, v = rnd((n, c.nkv, 64), seed + i, c.dev), rnd((n, c.nkv, 64), seed + 50 + i, c.dev, 1.0).float()
        k[:, :, 0] = 0
        k[0] = 0
        k[0, :, 0] = weight
        part = torch.arange(n, device=c.dev) * len(sizes) // n
        v *= torch.tensor(sizes, device=c.dev)[part][:, None, None]
        v[0] *= 0.02
        new = [0] * len(lens)
        new[i] = n
        c.append(k, v.half(), new)


def heavy_queries(t, nh, dev, seed):
    q = rnd((t, nh, 64), seed, dev)
    q[:, :, 0] = 8.0  # a score of 0.125 * 8 * weight on the first key
    return q


@pytest.mark.parametrize("sizes", [[1.0], [0.3], [0.1], [0.01], [0.001], [0.3, 0.001], [0.001, 0.3], [0.01, 300.0, 0.01]],
                         ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("new", [1, 3, 40, 300])
@pytest.mark.parametrize("total", [2048, 8192 + 64 + 37, 8192 + 5])
def test_weights_beside_a_heavy_first_key(cuda, sizes, new, total):
    """Most of the weight on one key of small value: what is left of the result are the many small weights."""
    c = Cache(1, 2, total, cuda)
    first_key_heavy(c, [total], sizes, 14.0, 3)
    q = heavy_queries(new, 8, cuda, 7)
    out = c.attend(q, [new], max_q=new)
    assert ops.paged_error() == 0
    check_weights(c, q, [new], out)


def test_weights_beside_a_heavy_first_key_mixed(cuda):
    lens, new = [3000, 700, 5000, 64, 129], [1, 200, 1, 3, 70]
    c = Cache(5, 2, 5000, cuda)
    first_key_heavy(c, lens, [0.03], 13.0, 3)
    q = heavy_queries(sum(new), 8, cuda, 7)
    out = c.attend(q, new)
    check_weights(c, q, new, out)


@pytest.mark.parametrize("late", [30, 64 + 30, 200])
@pytest.mark.parametrize("new", [2, 100, 400])
def test_small_values_before_large_ones(cuda, late, new):
    """The newest tokens' values are 300 times the others'; rows before them do not attend them, and their weights
    go by the values that they do attend."""
    for total in (1000, 1030, 1100, 64 * 17 + late):
        c = Cache(1, 2, total, cuda)
        k, v = rnd((total, 2, 64), 3, cuda), rnd((total, 2, 64), 4, cuda, 0.01)
        v[total - late:] *= 300
        c.append(k, v, [total])
        q = rnd((new, 8, 64), 7, cuda, 3.0)
        out = c.attend(q, [new], max_q=new)
        check_weights(c, q, [new], out)


@pytest.mark.parametrize("new", [1, 3, 70])
def test_page_scales_of_all_sizes(cuda, new):
    """Pages whose value scales go from fp16's smallest to large ones, in every order, and a tail beside them."""
    steps = [0.0, 3e-5, 1e-3, 0.0, 0.05, 2.0, 100.0, 5000.0, 60000.0]
    for sizes in (steps, steps[::-1], steps[4:] + steps[:4]):
        total = 64 * len(sizes) * 2 + 31
        c = Cache(1, 2, total, cuda)
        k, v = rnd((total, 2, 64), 3, cuda), rnd((total, 2, 64), 4, cuda).float().clamp(-1, 1)
        v[:-31] *= torch.tensor(sizes, device=cuda).repeat_interleave(64).repeat(2)[:, None, None]
        v[-31:] *= sizes[3]
        c.append(k, v.half(), [total])
        q = rnd((new, 8, 64), 7, cuda)
        out = c.attend(q, [new], max_q=new)
        assert bool(out.isfinite().all())
        check_weights(c, q, [new], out)


@pytest.mark.parametrize("new", [1, 2, 60])
def test_every_page_index_outside_the_pool_counts_as_absent(cuda, new):
    """Small negative numbers too, in every place of the table, beside a tail and without one."""
    for total in (500, 512):
        c = Cache(3, 2, 512, cuda)
        fill(c, [total] * 3, 3)
        q = rnd((3 * new, 8, 64), 7, cuda)
        want = c.attend(q, [new] * 3, max_q=new)
        assert ops.paged_error() == 0
        for wrong in (-2, -3, -4, -63, -64, c.kp8.shape[0], c.kp8.shape[0] + 1):
            for at in (0, 3, 5):  # (pages that all new rows attend in full)
                keep = int(c.table[1, at])
                c.table[1, at] = wrong
                out = c.attend(q, [new] * 3, max_q=new)
                assert ops.paged_error() == 2
                c.table[1, at] = keep
                assert torch.equal(out[:new], want[:new]) and torch.equal(out[2 * new:], want[2 * new:])
                k, v = (torch.cat([x[:, :64 * at], x[:, 64 * at + 64:]], 1) for x in (c.values(1, "k"), c.values(1, "v")))
                o, tol = plain_rows(q[new:2 * new], k, v, total - 64 - new, 0.125)
                close(out[new:2 * new], o, tol)


def well_formed(cu, rows):
    """Sequences whose two offsets are in range and in order and that begin at no less than every offset before."""
    top, ok = 0, []
    for s, (a, b) in enumerate(zip(cu, cu[1:])):
        top = max(top, min(max(a, 0), rows))
        if 0 <= a <= b <= rows and a >= top:
            ok.append(s)
    return ok


DISORDER = [[0, 800, 1000, 0, 1000], [0, 1000, 1001, 50, 60], [0, 1000, 1001, 0, 0], [500, 100, 200, 300], [900, 1001, 0],
            [0, 64, 63, 127, 200, 199, 500], [0, 2000, 10, 20], [-7, 30, 10, 900], [0, 100, 1500, 300, 400, 2**31 - 1],
            [1001, -2**31, 5, 9], [0, 0, 0, 300, 299, 299, 800], list(range(0, 600, 2)) + [3, 4, 700]]


@pytest.mark.parametrize("ctx", [0, 60, 640])
@pytest.mark.parametrize("cu", DISORDER, ids=lambda x: "-".join(map(str, x[:5])))
def test_append_offsets_out_of_order(cuda, cu, ctx):
    """A sequence that is out of order is skipped and reported; the others are appended, and no other page, scale or
    tail is touched."""
    rows, n = 1001, len(cu) - 1
    k, v = rnd((rows, 2, 64), 3, cuda), rnd((rows, 2, 64), 4, cuda)
    got, want = (Cache(n, 2, ctx + rows, cuda, seed=5) for _ in range(2))
    for c in (got, want):
        fill(c, [ctx] * n, 7)
    assert ops.paged_error() == 0
    for s in well_formed(cu, rows):
        a, b = cu[s], cu[s + 1]
        want.append(k[a:b], v[a:b], [b - a if i == s else 0 for i in range(n)])
        want.lens = [ctx] * n
    assert ops.paged_error() == 0
    ops.kv_paged_append(k, v, torch.tensor(cu, dtype=torch.int32, device=cuda), got.ints(), *got.t)
    assert ops.paged_error() == 4
    for x, y in zip(got.t, want.t):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("cu", [[0, 70], [-5, 20], [-5, 2], [20, 30, 51], [60, 70], [0, 20, 10, 40, 2**31 - 1], [-2**31, 50]],
                         ids=str)
def test_sequences_with_offsets_outside_are_skipped(cuda, cu):
    """Reported, and none of their rows written; the others as ever."""
    rows, n = 50, len(cu) - 1
    q, k, v = rnd((rows, 4, 64), 1, cuda), rnd((rows, 1, 64), 2, cuda), rnd((rows, 1, 64), 3, cuda)
    c = Cache(n, 1, 128, cuda)
    fill(c, [100] * n, 5)
    offsets = torch.tensor(cu, dtype=torch.int32, device=cuda)
    good = [(s, a, b) for s, (a, b) in enumerate(zip(cu, cu[1:])) if 0 <= a <= b <= rows]
    assert ops.paged_error() == 0
    calls = [(lambda out: ops.attn_varlen(q, k, v, offsets, out=out), lambda s, a, b: plain_rows(
        q[a:b], k[a:b].double().transpose(0, 1), v[a:b].double().transpose(0, 1), 0, 0.125))]
    calls += [(lambda out, m=m: ops.attn_paged(q, offsets, c.ints(), *c.t, max_q=m, out=out), lambda s, a, b: plain_rows(
        q[a:b], c.values(s, "k"), c.values(s, "v"), 100 - (b - a), 0.125)) for m in (None, 50)]
    for call, plain in calls:
        out = torch.full_like(q, 9.0)
        call(out)
        assert ops.paged_error() == 4
        for s, a, b in good:  # (a row that two of them claim is undefined)
            one = [sum(x <= r < y for _, x, y in good) == 1 for r in range(a, b)]
            o, tol = plain(s, a, b)
            close(out[a:b][one], o[one], tol[one])
        assert bool((out[[not any(x <= r < y for _, x, y in good) for r in range(rows)]] == 9).all())


def test_errors_are_seen_at_once_from_every_stream(cuda):
    """paged_error right after calls on side streams that are still waiting for their turn."""
    c = Cache(1, 1, 128, cuda)
    fill(c, [100], 5)
    q, one, bad, lens = rnd((1, 4, 64), 1, cuda), cum([1], cuda), cum([2], cuda), c.ints()
    table = torch.full_like(c.table, -1)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(streams[0]):
            torch.cuda._sleep(20_000_000)
            ops.attn_varlen(q, q[:, :1], q[:, :1], bad)
        with torch.cuda.stream(streams[1]):
            torch.cuda._sleep(40_000_000)
            ops.attn_paged(q, one, lens, table, *c.t[1:], max_q=1)
        assert ops.paged_error() == 6
        assert ops.paged_error() == 0


@pytest.mark.parametrize("bound", [61, 4096, 2**31 - 1, 2**31, 2**32, 2**32 + 1, 2**40])
def test_any_bound_of_the_longest_sequence(cuda, bound):
    """max_q is an upper bound, however large."""
    c = Cache(3, 2, 256, cuda)
    fill(c, [100, 200, 100], 3)
    q = rnd((62, 8, 64), 7, cuda)
    want = c.attend(q, [1, 60, 1], max_q=60)
    got = c.attend(q, [1, 60, 1], max_q=bound)
    assert ops.paged_error() == 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("nh,nkv", [(32, 8), (12, 4), (5, 1), (12, 1), (48, 1)])
def test_bits_go_by_the_sequence_alone(cuda, nh, nkv):
    """With the lengths and the keys the same, a sequence's bits depend neither on its neighbours' queries nor on what
    ran before."""
    lens, new = [400, 700, 352, 300], [150, 77, 129, 31]
    c = Cache(4, nkv, 700, cuda)
    fill(c, lens, 3)
    q = rnd((sum(new), nh, 64), 7, cuda, 2.0)
    big = rnd((900, nh, 64), 8, cuda, 40.0)
    kv = [rnd((sum(new), nkv, 64), 9 + i, cuda) for i in range(2)]
    calls = [lambda q: c.attend(q, new, max_q=max(new)), lambda q: ops.attn_varlen(q, *kv, cum(new, cuda))]
    for call in calls:
        want = call(q)
        for i in range(4):
            a, b = sum(new[:i]), sum(new[:i + 1])
            for scale in (0.0, 1.0, 30.0):
                other = q * scale
                other[a:b] = q[a:b]
                ops.attn_varlen(big * scale, big[:, :nkv], big[:, :nkv], cum([900], cuda))
                assert torch.equal(call(other)[a:b], want[a:b]), (i, scale)


@pytest.mark.parametrize("nh,nkv", [(32, 8), (5, 1), (12, 4)])
@pytest.mark.parametrize("new", [2, 3, 4, 100])
def test_bits_go_by_the_row_alone(cuda, nh, nkv, new):
    """The other new tokens' queries do not change a row's bits, whether its sequence is drafted tokens or a chunk."""
    c = Cache(1, nkv, 3000, cuda)
    fill(c, [2900], 3)
    q = rnd((new, nh, 64), 7, cuda, 2.0)
    kv = [rnd((new, nkv, 64), 9 + i, cuda) for i in range(2)]
    calls = [lambda q: c.attend(q, [new], max_q=new), lambda q: ops.attn_varlen(q, *kv, cum([new], cuda))]
    for call in calls:
        want = call(q)
        for row in (0, new // 2, new - 1):
            for scale in (0.0, 20.0):
                other = q * scale
                other[row] = q[row]
                assert torch.equal(call(other)[row], want[row]), (row, scale)
