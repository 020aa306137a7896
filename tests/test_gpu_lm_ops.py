"""The language-model operators on the GPU against plain 64-bit forms.

Tolerances count roundings.  H is half a step of the output type relative to
the value (bf16 2^-8, f16 2^-11, f32 2^-24, e4m3 2^-4), U = 2^-23 bounds one
fp32 operation with truncation, and a sum of n terms in any order is off by at
most n U times the sum of their magnitudes.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def vxb():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import vxb as V

    V.lib()
    return V


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half of a type's smallest step: what a rounding may cost below its normal
    range, where steps no longer shrink with the value (f16: 2^-24 / 2)."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, ref, tol, what=""):
    """|got - ref| <= tol element by element, non-finite values in the same places."""
    got = got.double()
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(got)), what + ": non-finite values differ"
    assert torch.equal(torch.isnan(ref), torch.isnan(got)), what + ": NaN differ"
    d = ((got - ref).abs() - tol)[fine]
    if d.numel():
        assert float(d.max()) <= 0, f"{what}: over the tolerance by {float(d.max()):.3e}"


# ---------------------------------------------------------------- rms norm --

def norm_case(vxb, N, C, dtype, res, out8, w32=False, pad=0, x=None, offset=0):
    def rows(seed, scale=1.0):  # rows of a wider matrix: stride C + pad, base `offset` elements in
        return randn(seed, N, C + pad + offset, dtype=dtype, scale=scale)[:, offset: offset + C]

    x = rows(1, 2.0) if x is None else x
    r = rows(2, 3.0) if res else None
    w = randn(3, C, dtype=torch.float32 if w32 else dtype, scale=0.2) + 1
    s = torch.full((N, C + pad), 7.0, dtype=dtype, device="cuda")[:, :C] if res else None
    kb = -(-C // 128)
    y = torch.empty(N, C + pad, dtype=F8 if out8 else dtype, device="cuda")[:, :C]
    sc = torch.full((N, kb), -1.0, device="cuda") if out8 else None
    vxb.rms_norm(x, w, y, y_scale=sc, residual=r, sum_out=s, eps=1e-5)
    h = x.double() + (r.double() if res else 0)
    ref = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5) * w.double()
    if res:  # x + residual in fp32, then one rounding
        close(s, h, h.abs() * (half_step(dtype) + U) + least(dtype), "sum")
    # the sum of squares: a thread adds 8 * 4 terms at most, then 10 levels of shuffles; the root halves its
    # error; rsqrtf 2 ulp, the division, eps, three products
    rel = (32 + 10) / 2 * U + 8 * U
    if not out8:
        close(y, ref, ref.abs() * (half_step(dtype) + rel) + least(dtype), "y")
        return
    top = torch.nn.functional.pad(ref, (0, kb * 128 - C)).view(N, kb, 128).abs().amax(2)
    close(sc, top / 448, top / 448 * (rel + 2 * U), "scale")
    by = sc.double().repeat_interleave(128, 1)[:, :C]
    # e4m3: half a step of the value, or half of the smallest step (2^-9) of the scale
    close(y.float().double() * by, ref, torch.maximum(ref.abs() * 2.0 ** -4, by * 2.0 ** -10) + ref.abs() * (rel + 4 * U),
          "codes")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,C", [(1, 1), (3, 7), (2, 8), (5, 128), (1, 1024), (33, 1000), (7, 1536), (4, 4096),
                                 (2, 4099), (3, 8192), (2, 16384), (1, 32768), (300, 200)])
@pytest.mark.parametrize("res,out8", [(False, False), (True, True)])
def test_rms_norm(vxb, N, C, dtype, res, out8):
    norm_case(vxb, N, C, dtype, res, out8)


@pytest.mark.parametrize("pad,offset", [(8, 0), (5, 0), (8, 8), (7, 1)])
def test_rms_norm_strided_rows(vxb, pad, offset):
    norm_case(vxb, 9, 640, torch.bfloat16, True, True, pad=pad, offset=offset)
    norm_case(vxb, 9, 640, torch.float32, True, False, pad=pad, offset=offset)
    norm_case(vxb, 9, 641, torch.float16, False, True, w32=True, pad=pad, offset=offset)


def test_rms_norm_in_place_and_zero_rows(vxb):
    x, r, w = randn(1, 6, 512, dtype=torch.bfloat16), randn(2, 6, 512, dtype=torch.bfloat16), torch.ones(512, device="cuda")
    x[2], r[2] = 0, 0
    a, b = torch.empty_like(x), torch.empty_like(x)
    vxb.rms_norm(x, w, a, residual=r, sum_out=b)
    y, s = x.clone(), r.clone()
    vxb.rms_norm(y, w, y, residual=s, sum_out=s)  # y over x, the sum over the residual
    assert torch.equal(y, a) and torch.equal(s, b) and not y[2].any()
    q, sc = torch.empty(6, 512, dtype=F8, device="cuda"), torch.empty(6, 4, device="cuda")
    vxb.rms_norm(x, w, q, y_scale=sc, residual=r)
    assert not q[2].float().any() and not sc[2].any() and sc[[0, 1, 3, 4, 5]].min() > 0


def test_rms_norm_zero_block_and_non_finite(vxb):
    x = randn(1, 5, 384, dtype=torch.float32)
    x[0, 128:256] = 0
    x[1, 5], x[2, 300], x[3, 0] = float("nan"), float("inf"), -float("inf")
    w = torch.ones(384, device="cuda")
    y = torch.empty_like(x)
    vxb.rms_norm(x, w, y)
    ref = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6)
    close(y, ref, ref.abs() * 64 * U, "y")
    q, sc = torch.empty(5, 384, dtype=F8, device="cuda"), torch.empty(5, 3, device="cuda")
    vxb.rms_norm(x, w, q, y_scale=sc)
    assert sc[0, 1] == 0 and not q[0, 128:256].float().any()
    v = q.float() * sc.repeat_interleave(128, 1)
    assert torch.isfinite(v[0]).all() and torch.isfinite(v[4]).all()
    assert torch.isnan(v[1]).all() and torch.isnan(v[2, 300]) and torch.isnan(v[3, 0])


# ------------------------------------------------------------- fp8 product --

def codes(seed, rows, K, block_rows, spread=0.5):
    """Quantised matrix and its scales: blocks of unlike size."""
    v = randn(seed, rows, K) * torch.exp(spread * randn(seed + 1, K))
    kb, rb = -(-K // 128), -(-rows // block_rows)
    p = torch.zeros(rb * block_rows, kb * 128, device="cuda")
    p[:rows, :K] = v
    s = p.view(rb, block_rows, kb, 128).abs().amax(dim=(1, 3)) / 448
    by = s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :K]
    return (v / by).to(F8), s


def wide(t, stride, offset=0):
    """The same matrix as rows of a wider buffer."""
    b = torch.zeros(t.shape[0], stride + offset, dtype=torch.uint8, device="cuda").view(t.dtype) \
        if t.dtype == F8 else torch.zeros(t.shape[0], stride + offset, dtype=t.dtype, device="cuda")
    v = b[:, offset: offset + t.shape[1]]
    v.copy_(t)
    return v


def product_ref(x, xs, w, ws, bias):
    K, M = x.shape[1], w.shape[0]
    xd = x.float().double() * xs.double().repeat_interleave(128, 1)[:, :K]
    wd = w.float().double() * ws.double().repeat_interleave(128, 0)[:M].repeat_interleave(128, 1)[:, :K]
    b = 0 if bias is None else bias.double()
    return xd @ wd.t() + b, xd.abs() @ wd.abs().t() + (0 if bias is None else b.abs())


def product_tol(ref, mag, K, dtype):
    # a sum of K terms, a scaling and an addition for each block, the bias; then the output's rounding
    return mag * (K + 2 * (-(-K // 128)) + 2) * U + ref.abs() * half_step(dtype) + 2.0 ** -25


def product_case(vxb, N, K, M, dtype, bias=True):
    x, xs = codes(1, N, K, 1)
    w, ws = codes(5, M, K, 128)
    b = randn(9, M) if bias else None
    y = torch.full((N, M), float("nan"), dtype=dtype, device="cuda")
    vxb.fp8_product(x, xs, w, ws, y, bias=b)
    ref, mag = product_ref(x, xs, w, ws, b)
    close(y, ref, product_tol(ref, mag, K, dtype), f"{N}x{K}x{M}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,M", [
    (1, 16, 1), (1, 128, 128), (2, 1024, 64), (16, 1536, 1000), (17, 144, 129), (31, 4096, 512), (33, 2048, 255),
    (64, 8192, 384), (65, 128, 64), (77, 1536, 1001), (128, 1008, 256), (129, 256, 130), (200, 4096, 1024),
    (1, 8192, 8192), (1, 4096, 4096), (1, 1040, 4099), (2, 2048, 129), (2, 16, 3), (3, 528, 70), (700, 512, 7000), (2500, 384, 2056), (1281, 640, 4100)])
def test_fp8_product(vxb, N, K, M, dtype):
    product_case(vxb, N, K, M, dtype)


def test_fp8_product_types_and_bias(vxb):
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        product_case(vxb, 5, 512, 300, dtype, bias=False)
        product_case(vxb, 150, 512, 300, dtype, bias=True)


@pytest.mark.parametrize("N", [1, 2, 3, 50, 150])
def test_fp8_product_strided(vxb, N):
    K, M = 400, 200
    x, xs = codes(1, N, K, 1)
    w, ws = codes(5, M, K, 128)
    y = torch.full((N, M + 9), 3.0, device="cuda")
    vxb.fp8_product(wide(x, 448, 32), wide(xs, 7, 2), wide(w, 512, 16), ws, y[:, 5: 5 + M])
    ref, mag = product_ref(x, xs, w, ws, None)
    close(y[:, 5: 5 + M], ref, product_tol(ref, mag, K, torch.float32))
    assert (y[:, :5] == 3).all() and (y[:, 5 + M:] == 3).all()  # what lies beside the output stays


def test_fp8_product_non_finite_stays_in_its_row_and_column(vxb):
    for N in (20, 140):
        x, xs = codes(1, N, 512, 1)
        w, ws = codes(5, 260, 512, 128)
        xs[3, 1] = float("inf")
        x.view(torch.uint8)[7, 300] = 0x7F  # NaN
        w.view(torch.uint8)[150, 20] = 0x7F
        y = torch.empty(N, 260, device="cuda")
        vxb.fp8_product(x, xs, w, ws, y)
        bad = torch.zeros(N, 260, dtype=torch.bool, device="cuda")
        bad[3], bad[7], bad[:, 150] = True, True, True
        assert torch.equal(~torch.isfinite(y), bad)


def test_fp8_product_of_one_token_with_non_finite_codes(vxb):
    x, xs = codes(1, 2, 512, 1)
    w, ws = codes(5, 260, 512, 128)
    x.view(torch.uint8)[1, 300] = 0xFF  # NaN
    w.view(torch.uint8)[150, 20] = 0x7F
    ws[0, 2] = float("inf")
    y = torch.empty(2, 260, device="cuda")
    vxb.fp8_product(x, xs, w, ws, y)
    bad = torch.zeros(2, 260, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 150], bad[:, :128] = True, True, True
    assert torch.equal(~torch.isfinite(y), bad)


def test_fp8_product_repeats_bit_for_bit(vxb):
    for N, K, M in ((1, 1024, 700), (7, 4096, 640), (100, 2048, 640), (600, 1024, 2000)):
        x, xs = codes(1, N, K, 1)
        w, ws = codes(5, M, K, 128)
        a, b = (torch.empty(N, M, device="cuda") for _ in range(2))
        vxb.fp8_product(x, xs, w, ws, a)
        for _ in range(5):
            vxb.fp8_product(x, xs, w, ws, b)
            assert torch.equal(a, b)


# ------------------------------------------------------------------ rotary --

def turned(v, pos, inv, factor, inter):
    """64-bit rotation and the sum of its magnitudes."""
    R = 2 * inv.shape[0]
    ang = pos.double()[:, None, None] * inv.double()
    c, s = ang.cos() * factor, ang.sin() * factor
    v = v.double()
    a, b = (v[..., 0:R:2], v[..., 1:R:2]) if inter else (v[..., :R // 2], v[..., R // 2:R])
    x, y, mag = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * factor
    join = (lambda p, q: torch.stack((p, q), -1).flatten(-2)) if inter else (lambda p, q: torch.cat((p, q), -1))
    rest = v[..., R:]
    return torch.cat((join(x, y), rest), -1), torch.cat((join(mag, mag), torch.zeros_like(rest)), -1)


def rotary_tol(ref, mag, dtype, R):
    # the turn is rounded to fp32 (half of 2^-24 turns: 2^-25 * 2 pi rad), cos and sin are off by 2 ulp, times the
    # factor, a product and a sum each
    return mag * (2.0 ** -25 * 2 * math.pi + 6 * U) + ref.abs() * half_step(dtype) * (mag > 0) + 2.0 ** -25 * (mag > 0)


ROTARY = [  # N, Hq, Hk, D, R
    (1, 1, 1, 2, 2), (5, 4, 2, 64, 64), (3, 16, 2, 64, 32), (257, 7, 1, 128, 128), (40, 32, 8, 128, 64),
    (9, 3, 3, 80, 40), (6, 2, 2, 20, 6), (2000, 4, 2, 96, 96), (11, 2, 1, 300, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("N,Hq,Hk,D,R", ROTARY)
def test_rotary(vxb, N, Hq, Hk, D, R, inter, dtype):
    q, k = randn(1, N, Hq, D, dtype=dtype), randn(2, N, Hk, D, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    pos = torch.randint(0, 3000000, (N,), generator=g, device="cuda")
    pos[0] = 0
    f, factor = vxb.rotary_frequencies(R, factors=np.linspace(1, 30, R // 2), original_length=4096, length=100000)
    inv = torch.from_numpy(f).cuda()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    vxb.rotary(q, pos, inv, qo, k=k, k_out=ko, interleaved=inter, factor=factor)
    for out, v in ((qo, q), (ko, k)):
        ref, mag = turned(v, pos, inv, factor, inter)
        close(out, ref, rotary_tol(ref, mag, dtype, R))
    vxb.rotary(q, pos, inv, q, k=k, k_out=k, interleaved=inter, factor=factor)  # in place
    assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("order", ["slots first", "heads first", "joint"])
@pytest.mark.parametrize("dt,D,R,page", [(torch.bfloat16, 64, 48, 16), (torch.float32, 64, 64, 16),
                                         (torch.float16, 20, 10, 10), (torch.float32, 6, 2, 1)])
def test_rotary_append(vxb, inter, order, dt, D, R, page):
    N, Hq, Hk, pages = 50, 8, 2, 9 if page > 1 else 140
    qkv = randn(1, N, (Hq + 2 * Hk) * D, dtype=dt)  # rows of one projection
    q, k, v = (t.view(N, -1, D) for t in qkv.split([Hq * D, Hk * D, Hk * D], 1))
    if order == "heads first":
        kc, vc = (randn(s, pages, Hk, page, D, dtype=dt).transpose(1, 2) for s in (4, 5))
    elif order == "joint":
        both = randn(4, pages, 2, page, Hk, D, dtype=dt)
        kc, vc = both[:, 0], both[:, 1]
    else:
        kc, vc = (randn(s, pages, page, Hk, D, dtype=dt) for s in (4, 5))
    g = torch.Generator(device="cuda").manual_seed(6)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:N].contiguous()
    slots[7], slots[11], slots[13] = -1, pages * page, 1 << 60  # padding tokens
    pos = torch.arange(100, 100 + N, device="cuda")
    inv = torch.from_numpy(vxb.rotary_frequencies(R)[0]).cuda()
    rk, rv = kc.double().flatten(0, 1), vc.double().flatten(0, 1)
    tk = torch.zeros_like(rk)
    keep = (slots >= 0) & (slots < pages * page)
    ref, mag = turned(k, pos, inv, 1.0, inter)
    rk[slots[keep]], tk[slots[keep]] = ref[keep], rotary_tol(ref, mag, dt, R)[keep]
    rv[slots[keep]] = v.double()[keep]
    qo = torch.empty(N, Hq, D, dtype=dt, device="cuda")
    vxb.rotary_append(q, k, v, pos, slots, inv, qo, kc, vc, interleaved=inter)
    close(kc.double().flatten(0, 1), rk, tk, "k_cache")
    assert torch.equal(vc.double().flatten(0, 1), rv)
    ref, mag = turned(q, pos, inv, 1.0, inter)
    close(qo, ref, rotary_tol(ref, mag, dt, R), "q")


# --------------------------------------------------------- paged attention --

class Batch:
    """Ragged sequences over shuffled pages; places that no token sees hold NaN."""

    def __init__(self, q_len, kv_len, Hq, Hk, D, page, dtype, window=0, seed=0, order="slots first", tail=0,
                 max_pages=None):
        self.q_len, self.kv_len, self.window, self.page, self.D = q_len, kv_len, window, page, D
        self.Hq, self.Hk, self.dtype = Hq, Hk, dtype
        B, N = len(q_len), sum(q_len)
        used = [-(-n // page) for n in kv_len]
        pages = sum(used) + 3
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(pages, generator=g).tolist()
        width = max_pages or max(used + [1])
        table = torch.randint(-5, pages + 5, (B, width), generator=g)  # what lies past a sequence's pages is anything
        shape = (pages, Hk, page, D) if order == "heads first" else (pages, page, Hk, D)
        self.k = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        self.v = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        if order == "heads first":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.keys, at = [], 0
        for b, n in enumerate(used):
            mine = perm[at: at + n]
            at += n
            table[b, :n] = torch.tensor(mine, dtype=table.dtype)
            kk, vv = (randn(seed + 10 * b + i, kv_len[b], Hk, D, dtype=dtype) for i in (1, 2))
            for p, pg in enumerate(mine):
                m = min(page, kv_len[b] - p * page)
                self.k[pg, :m] = kk[p * page: p * page + m]
                self.v[pg, :m] = vv[p * page: p * page + m]
            self.keys.append((kk, vv))
        self.table = table.to(torch.int32).cuda()
        self.cu = torch.tensor([0] + list(np.cumsum(q_len)), dtype=torch.int32, device="cuda")
        self.kv = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
        self.q = randn(seed + 3, N + tail, Hq, D, dtype=dtype)
        self.out = torch.full((N + tail, Hq, D), 5.0, dtype=dtype, device="cuda")

    def run(self, vxb, **kw):
        vxb.paged_attention(self.q, self.k, self.v, self.table, self.cu, self.kv, self.out, window=self.window, **kw)
        return self.out

    def check(self, hidden=None, scale=None):
        """Against softmax(q k^T) v in 64 bits; hidden(b) -> extra mask of keys [kv]."""
        scale = self.D ** -0.5 if scale is None else scale
        G, at = self.Hq // self.Hk, 0
        h = half_step(self.dtype)
        for b, (n, kv) in enumerate(zip(self.q_len, self.kv_len)):
            if not n:
                continue
            q = self.q[at: at + n].double()
            k, v = (t.double().repeat_interleave(G, 1) for t in self.keys[b])
            pos = torch.arange(kv - n, kv, device="cuda")[:, None]
            key = torch.arange(kv, device="cuda")[None]
            seen = key <= pos
            if self.window:
                seen = seen & (key > pos - self.window)
            if hidden is not None:
                seen = seen & ~hidden(b)[None]
            s = torch.einsum("qhd,khd->hqk", q, k) * scale
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True) if kv else torch.zeros(self.Hq, n, 1, dtype=torch.float64, device="cuda")
            p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
            p = torch.where(seen, p, torch.zeros_like(p))
            w = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            # a value that a token does not see has no weight, whatever it is
            ref = torch.einsum("hqk,khd->qhd", w, torch.nan_to_num(v, 0, 0, 0))
            mag = torch.einsum("hqk,khd->qhd", w, torch.nan_to_num(v, 0, 0, 0).abs())
            odd = ~torch.isfinite(v)
            if odd.any():
                mark = torch.einsum("qk,khd->qhd", seen.double(), odd.double()) > 0
                ref = torch.where(mark, torch.full_like(ref, math.nan), ref)
            # a score is a sum of D products, scaled (its error is its weight's, relative); the sums run over
            # kv keys; a weight is rounded to the type, the exponential is off by 2 ulp of fp32 at arguments
            # whose rounding adds |s| U
            big = torch.einsum("qhd,khd->hqk", q.abs(), torch.nan_to_num(k, 0, 0, 0).abs())
            big = float((big * scale).max()) if kv else 0.0
            rel = h + 2 * (self.D * U * big + 4 * U * big) + (kv + 20) * U
            got = self.out[at: at + n].double()
            if odd.any():
                assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), "non-finite values reach other rows"
                got = torch.where(torch.isfinite(ref), got, ref)
            close(got, ref, mag * rel + ref.abs() * h + 1e-7, f"sequence {b}")
            at += n
        assert (self.out[at:] == 5.0).all(), "rows behind the last sequence changed"


DECODE = [  # q_len, kv_len, Hq, Hk, D, page
    ([1], [1], 1, 1, 64, 16), ([1, 1, 1], [1, 17, 64], 16, 2, 64, 16), ([1] * 5, [130, 1, 63, 65, 1000], 32, 8, 128, 64),
    ([1, 0, 1], [5, 9, 0], 7, 1, 80, 32), ([1], [5000], 32, 8, 128, 64), ([1, 1], [3000, 10], 28, 4, 128, 128),
    ([1], [2049], 64, 2, 96, 16), ([1, 1], [777, 256], 48, 1, 64, 256), ([1] * 40, list(range(1, 41)), 4, 4, 8, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", DECODE, ids=str)
def test_attention_single_tokens(vxb, case, dtype):
    b = Batch(*case, dtype)
    b.run(vxb)
    b.check()


CHUNKS = [  # q_len, kv_len, Hq, Hk, D, page
    ([2], [2], 4, 4, 64, 16), ([37, 5, 1], [1000, 5, 300], 16, 2, 64, 16), ([130], [130], 8, 2, 128, 64),
    ([300, 0, 7, 129], [700, 33, 7, 129], 7, 1, 128, 32), ([65], [4100], 14, 2, 80, 16), ([513], [600], 4, 2, 96, 128),
    ([16, 3], [16, 2000], 40, 1, 128, 16), ([260], [1500], 2, 1, 128, 256), ([50, 90], [50, 900], 200, 1, 64, 32),
    ([200, 1, 0, 64], [2000, 900, 7, 6000], 12, 4, 128, 64),
    ([9 + b % 3 for b in range(300)], [20 + 7 * b % 90 for b in range(300)], 8, 1, 64, 16), ([3, 4], [2, 1], 4, 2, 64, 16), ([256], [1024], 2, 2, 40, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 1, 50, 100000])
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: str(c)[:60])
def test_attention_chunks(vxb, case, window, dtype):
    b = Batch(*case, dtype, window=window, tail=3)
    b.run(vxb)
    b.check()


def test_attention_heads_first_cache_wide_table_and_strided_rows(vxb):
    b = Batch([20, 1, 1], [300, 40, 5], 8, 2, 64, 16, torch.bfloat16, order="heads first", max_pages=50)
    qkv = torch.zeros(22, 12, 64, dtype=torch.bfloat16, device="cuda")
    qkv[:, 2:10] = b.q
    b.q = qkv[:, 2:10]
    wide_out = torch.full((22, 9, 72), 5.0, dtype=torch.bfloat16, device="cuda")
    b.out = wide_out[:, 1:, :64]
    b.run(vxb)
    b.check()
    assert (wide_out[:, 0] == 5).all() and (wide_out[..., 64:] == 5).all()


@pytest.mark.parametrize("q_len", [5, 150])
def test_attention_scale_and_zero_scale(vxb, q_len):
    for scale in (0.0, 1.0, -0.3):
        b = Batch([q_len, 1], [q_len + 85, 33], 4, 2, 64, 16, torch.float16)
        b.run(vxb, scale=scale)
        b.check(scale=scale)


@pytest.mark.parametrize("q_len", [1, 60, 200])
def test_attention_absent_pages(vxb, q_len):
    """Pages given back (entries outside the cache) leave their keys unseen; a token all of whose keys are gone gets zeros."""
    page, kv = 16, 320
    b = Batch([q_len, q_len], [kv, kv], 8, 2, 64, page, torch.bfloat16, window=64)
    gone = [torch.zeros(kv, dtype=torch.bool, device="cuda") for _ in range(2)]
    for p, entry in ((0, -1), (7, 1 << 30), (18, -7)):
        b.table[0, p] = entry
        gone[0][p * page: (p + 1) * page] = True
    b.table[1, :] = -1
    gone[1][:] = True
    b.run(vxb)
    b.check(hidden=lambda i: gone[i])
    assert not b.out[q_len:].any()


@pytest.mark.parametrize("q_len,kv,window,D", [(40, 200, 0, 64), (40, 200, 30, 128), (200, 200, 0, 128), (3, 70, 10, 64),
                                               (300, 900, 100, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_non_finite_values_reach_only_tokens_that_see_them(vxb, q_len, kv, window, D, value):
    b = Batch([q_len], [kv], 8, 2, D, 16, torch.bfloat16, window=window)
    for j, d in ((kv - 1, 3), (kv - q_len // 2 - 1, 20), (kv - q_len + 1, 8)):
        pg = int(b.table[0, j // 16])
        b.v[pg, j % 16, 1, d] = value
        b.keys[0][1][j, 1, d] = value
    b.run(vxb)
    b.check()


def test_attention_non_finite_keys_reach_only_tokens_that_see_them(vxb):
    b = Batch([30], [100], 4, 2, 64, 16, torch.float16)
    pg = int(b.table[0, 90 // 16])
    b.k[pg, 90 % 16, 0, 5] = float("nan")
    b.run(vxb)
    bad = ~torch.isfinite(b.out).all(-1)  # [token, head]: tokens from position 90 on, heads of key head 0
    want = torch.zeros(30, 4, dtype=torch.bool, device="cuda")
    want[20:, :2] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("q_len", [[1, 1, 1], [30, 1, 9], [200, 70, 90]])
def test_attention_rows_before_the_first_sequence_and_shared_pages(vxb, q_len):
    """Sequences may start behind row 0 of q, and may share pages (a common prompt)."""
    b = Batch(q_len, [n + 64 for n in q_len], 8, 2, 64, 16, torch.bfloat16)
    for i in (1, 2):  # the first 48 keys are sequence 0's
        b.table[i, :3] = b.table[0, :3]
        for x in (0, 1):
            b.keys[i][x][:48] = b.keys[0][x][:48]
    b.run(vxb)
    b.check()
    ref = b.out.clone()
    b.q = torch.cat([randn(9, 5, 8, 64, dtype=torch.bfloat16), b.q])
    b.out = torch.full_like(b.q, 5.0)
    b.cu += 5
    b.run(vxb)
    assert torch.equal(b.out[5:], ref) and (b.out[:5] == 5).all()


def test_calls_on_no_rows(vxb):
    e = lambda *s, d=torch.bfloat16: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    vxb.rms_norm(e(0, 64), e(64), e(0, 64))
    vxb.fp8_product(e(0, 64, d=F8), e(0, 1, d=torch.float32), e(5, 64, d=F8), e(1, 1, d=torch.float32), e(0, 5))
    q, k, c, pos, f = e(0, 4, 64), e(0, 2, 64), e(3, 16, 2, 64), e(0, d=torch.int64), e(32, d=torch.float32)
    vxb.rotary(q, pos, f, q)
    vxb.rotary_append(q, k, k, pos, pos, f, q, c, c)
    vxb.paged_attention(q, c, c, i(0, 0).view(1, 2), i(0, 0), i(9), q)
    one, table = randn(1, 1, 4, 64, dtype=torch.bfloat16), e(0, 2, d=torch.int32)
    out = torch.full_like(one, 5.0)
    vxb.paged_attention(one, c, c, table, i(0), i(), out)  # no sequences: every row is outside
    torch.cuda.synchronize()
    assert (out == 5).all()


@pytest.mark.parametrize("q_len", [1, 200])
def test_attention_without_pages_or_keys(vxb, q_len):
    """A cache of no pages, tables of no entries: every token sees nothing and gets zeros."""
    q = randn(1, q_len, 8, 64, dtype=torch.bfloat16)
    c = torch.empty(0, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for table in (i(0, 1).view(1, 2), torch.empty(1, 0, dtype=torch.int32, device="cuda")):
        out = torch.full_like(q, 5.0)
        vxb.paged_attention(q, c, c, table, i(0, q_len), i(30), out)
        assert not out.any()


def test_attention_lengths_out_of_range_are_cut(vxb):
    """kv_len beyond the table's pages counts as the table's capacity; rows outside q are not there."""
    b = Batch([1, 1], [64, 64], 4, 2, 64, 16, torch.bfloat16)
    b.run(vxb)
    ref = b.out.clone()
    b.kv[0] = 1 << 30
    b.run(vxb)
    assert torch.equal(b.out, ref)
    b.kv[1], b.out[1] = -5, 5
    b.run(vxb)
    assert torch.equal(b.out[0], ref[0]) and not b.out[1].any()
    b.kv[1] = 64
    b.cu[2] = 900  # past q: the sequence is left out
    b.out[1] = 5
    b.run(vxb)
    assert torch.equal(b.out[0], ref[0]) and (b.out[1] == 5).all()


@pytest.mark.parametrize("q_len", [6, 100])
def test_attention_widest_window_is_none(vxb, q_len):
    """Fewer keys than new tokens: the first tokens stand before key 0, and a window of 2^31 - 1
    reaches no further than any other."""
    b = Batch([q_len], [q_len - 4], 8, 2, 64, 16, torch.bfloat16)
    b.run(vxb)
    b.check()
    ref = b.out.clone()
    for window in (2 ** 31 - 1, 2 ** 30, b.table.shape[1] * 16):
        b.window = window
        b.out.fill_(5.0)
        b.run(vxb)
        assert torch.equal(b.out, ref)


@pytest.mark.parametrize("heads", [1, 8])
def test_attention_row_ranges_that_overlap_stay_in_bounds(vxb, heads):
    """Not sequences, so their rows' values mean nothing; the rows of proper ones and those of none do."""
    b = Batch([40, 20, 20, 20], [60, 50, 45, 70], heads, 1, 64, 16, torch.bfloat16, tail=4)
    b.cu[2] = 30  # the second ends before it starts, the third begins inside the first
    b.run(vxb)
    torch.cuda.synchronize()
    assert torch.isfinite(b.out).all() and (b.out[100:] == 5).all()


def test_axes_of_one_element_have_any_stride(vxb):
    b = Batch([1], [40], 4, 1, 64, 16, torch.bfloat16)
    b.k, b.v = (t.as_strided(t.shape, (t.stride(0), t.stride(1), 3, 1)) for t in (b.k, b.v))
    b.q = b.q.as_strided(b.q.shape, (7, b.q.stride(1), 1))
    b.run(vxb)
    b.check()


@pytest.mark.parametrize("q_len", [1, 100])
def test_attention_offsets_beyond_32_bits(vxb, q_len):
    """A cache of 2.2e9 elements; the pages in use are its first and last."""
    page, Hk, D = 64, 8, 128
    pages = 2_200_000_000 // (page * Hk * D)
    free, _ = torch.cuda.mem_get_info()
    if free < 12e9:
        pytest.skip("needs 12 GB")
    b = Batch([q_len], [4 * page - 5], 16, Hk, D, page, torch.bfloat16)
    k, v = (torch.empty(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = [pages - 1, 0, pages - 2, 1]
    for i, p in enumerate(at):
        k[p], v[p] = b.k[int(b.table[0, i])], b.v[int(b.table[0, i])]
    b.k, b.v = k, v
    b.table = torch.tensor([at], dtype=torch.int32, device="cuda")
    b.run(vxb)
    b.check()
    slots = torch.tensor([(pages - 1) * page + 3, 5], device="cuda")
    kk, pos = randn(1, 2, Hk, D, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64, device="cuda")
    inv = torch.from_numpy(vxb.rotary_frequencies(D)[0]).cuda()
    vxb.rotary_append(kk, kk, kk, pos, slots, inv, torch.empty_like(kk), k, v)
    assert torch.equal(v[pages - 1, 3], kk[0]) and torch.equal(k[0, 5], kk[1])


# ------------------------------------------------------ streams and graphs --

def test_operators_on_another_stream(vxb):
    b = Batch([1, 1], [3000, 5000], 32, 8, 128, 64, torch.bfloat16)
    b.run(vxb)
    torch.cuda.synchronize()
    ref = b.out.clone()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream, torch.cuda.default_stream(), 0):
        b.out.fill_(5.0)
        s.wait_stream(torch.cuda.current_stream())
        b.run(vxb, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(b.out, ref)


def test_products_and_norms_on_two_streams_at_once(vxb):
    """Calls that share the device keep apart: clusters, tensor memory and staging are their own."""
    sets = []
    for i, (N, K, M) in enumerate(((9, 4096, 512), (600, 1024, 2000), (200, 2048, 640), (3000, 512, 1536))):
        x, xs = codes(10 * i, N, K, 1)
        w, ws = codes(10 * i + 5, M, K, 128)
        y = torch.empty(N, M, dtype=torch.bfloat16, device="cuda")
        vxb.fp8_product(x, xs, w, ws, y)
        n = torch.empty_like(y)
        vxb.rms_norm(y, torch.ones(M, device="cuda"), n)
        sets.append((x, xs, w, ws, torch.ones(M, device="cuda"), y.clone(), n.clone(), torch.empty_like(y), torch.empty_like(n)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(8):
        for i, (x, xs, w, ws, g, ry, rn, y, n) in enumerate(sets):
            st = streams[(i + turn // 4) % 2]
            st.wait_stream(streams[(i + turn // 4 + 1) % 2] if turn % 4 == 0 else st)
            vxb.fp8_product(x, xs, w, ws, y, stream=st)
            vxb.rms_norm(y, g, n, stream=st)
    torch.cuda.synchronize()
    for x, xs, w, ws, g, ry, rn, y, n in sets:
        assert torch.equal(y, ry) and torch.equal(n, rn)


def test_two_captured_graphs_and_an_eager_call(vxb):
    """Graphs captured one after the other keep their own workspaces: replayed
    on two streams with an eager call between, each gives its own answer."""
    bs = [Batch([1], [4000 + 500 * i], 32, 8, 128, 64, torch.bfloat16, seed=100 * i) for i in range(3)]
    refs = []
    for b in bs:
        refs.append(b.run(vxb).clone())
    graphs = []
    for b in bs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run(vxb)
        graphs.append(g)
    for b in bs:
        b.out.fill_(5.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        bs[2].run(vxb)
    torch.cuda.synchronize()
    for b, r in zip(bs, refs):
        assert torch.equal(b.out, r)


def test_given_workspace_must_be_large_enough(vxb):
    b = Batch([1], [5000], 32, 8, 128, 64, torch.bfloat16)
    need = vxb.lib().vxb_paged_attention_workspace(1, 1, 32, 8, 128, b.table.shape[1], 64)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    b.run(vxb, workspace=ws)
    b.check()
    if need:
        with pytest.raises(vxb.VxbError) as e:
            b.run(vxb, workspace=ws[: need - 1])
        assert e.value.code == vxb.ERR_INVALID_ARGUMENT


# ------------------------------------------------------- a layer, as it runs --

def test_streaming_layer_feeds_the_decoder(vxb):
    """Norm -> 8-bit product -> rotary and cache -> attention -> 8-bit product for a
    prompt chunk and then single tokens of two streams, the last product writing
    the fp32 latents that the audio decoder reads on the same stream; every step
    captured into one graph.  Against the same layer in 64 bits, which takes over
    the quantised operands (their codes are what the kernels multiply)."""
    from models import model_path

    bf = torch.bfloat16
    B, C, Hq, Hk, D, page, T = 2, 256, 8, 2, 32, 16, 6
    wqkv, wqkv_s = codes(11, (Hq + 2 * Hk) * D, C, 128, spread=0.0)
    wqkv_s = wqkv_s * 0.06
    wo, wo_s = codes(21, 64 * T, Hq * D, 128, spread=0.0)
    wo_s = wo_s * 0.06
    gain, gain2 = 1 + randn(31, C, scale=0.1, dtype=bf), torch.ones(Hq * D, dtype=bf, device="cuda")
    inv = torch.from_numpy(vxb.rotary_frequencies(D)[0]).cuda()
    kc, vc = (torch.zeros(8, page, Hk, D, dtype=bf, device="cuda") for _ in range(2))
    table = torch.tensor([[3, 1, 6], [0, 5, 2]], dtype=torch.int32, device="cuda")

    def buffers(N):
        e = lambda *s, d=bf: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
        return dict(h8=e(N, C, d=F8), hs=e(N, C // 128, d=torch.float32), sum=e(N, C), qkv=e(N, (Hq + 2 * Hk) * D),
                    q=e(N, Hq, D), o=e(N, Hq, D), o8=e(N, Hq * D, d=F8), os=e(N, Hq * D // 128, d=torch.float32),
                    z=e(N, 64 * T, d=torch.float32))

    def layer(x, res, pos, slots, cu, kv, w):
        N = x.shape[0]
        vxb.rms_norm(x, gain, w["h8"], y_scale=w["hs"], residual=res, sum_out=w["sum"])
        vxb.fp8_product(w["h8"], w["hs"], wqkv, wqkv_s, w["qkv"])
        q, k, v = (t.view(N, -1, D) for t in w["qkv"].split([Hq * D, Hk * D, Hk * D], 1))
        vxb.rotary_append(q, k, v, pos, slots, inv, w["q"], kc, vc)
        vxb.paged_attention(w["q"], kc, vc, table, cu, kv, w["o"])
        vxb.rms_norm(w["o"].view(N, Hq * D), gain2, w["o8"], y_scale=w["os"])
        vxb.fp8_product(w["o8"], w["os"], wo, wo_s, w["z"])

    history = [[], []]  # per stream: (k, v) in 64 bits, from the rounded projection

    def check(pos, seq, w):
        ref, mag = product_ref(w["h8"], w["hs"], wqkv, wqkv_s, None)
        close(w["qkv"], ref, product_tol(ref, mag, C, bf), "qkv")
        q, k, v = (t.view(len(seq), -1, D) for t in w["qkv"].split([Hq * D, Hk * D, Hk * D], 1))
        k64, mk = turned(k, pos, inv, 1.0, False)
        q64, mq = turned(q, pos, inv, 1.0, False)
        close(w["q"], q64, rotary_tol(q64, mq, bf, D), "q")
        for i, b in enumerate(seq):
            history[b].append((k64[i].to(bf).double(), v[i].double()))
            kk, vv = (torch.stack(t).repeat_interleave(Hq // Hk, 1) for t in zip(*history[b]))
            s = torch.einsum("hd,khd->hk", w["q"][i].double(), kk) * D ** -0.5
            p = torch.softmax(s, -1)
            ref, mag = torch.einsum("hk,khd->hd", p, vv), torch.einsum("hk,khd->hd", p, vv.abs())
            # a key of the cache may lie one rounding of bf16 beside the reference's (2^-7 of it): the scores'
            # error is their weights', relative
            big = float((torch.einsum("hd,khd->hk", w["q"][i].double().abs(), kk.abs()) * D ** -0.5).max())
            close(w["o"][i], ref, mag * (2 * 2.0 ** -7 * big + 2 * half_step(bf)) + 1e-6, "attention")
        ref, mag = product_ref(w["o8"], w["os"], wo, wo_s, None)
        close(w["z"], ref, product_tol(ref, mag, Hq * D, torch.float32), "latents")

    def slot_of(b, p):
        return int(table[b, p // page]) * page + p % page

    lens = [21, 17]
    seq = [b for b in range(B) for _ in range(lens[b])]
    at = [p for b in range(B) for p in range(lens[b])]
    N = len(seq)
    w = buffers(N)
    pos = torch.tensor(at, device="cuda")
    slots = torch.tensor([slot_of(b, p) for b, p in zip(seq, at)], device="cuda")
    cu = torch.tensor([0, lens[0], N], dtype=torch.int32, device="cuda")
    layer(randn(41, N, C, dtype=bf), randn(42, N, C, dtype=bf), pos, slots, cu,
          torch.tensor(lens, dtype=torch.int32, device="cuda"), w)
    check(pos, seq, w)

    # single tokens: one graph, its inputs changed between replays; the decoder runs on what it left
    path, _ = model_path(quant="q4_0", seed=0)
    d = vxb.Decoder(0)
    d.load_gguf(path)
    d.prepare()
    d.build_plan(B, T)
    w = buffers(B)
    x, res = torch.empty(B, C, dtype=bf, device="cuda"), torch.empty(B, C, dtype=bf, device="cuda")
    pos, slots = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.full((B,), -1, device="cuda")
    cu, kv = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
    x.zero_(), res.zero_()
    layer(x, res, pos, slots, cu, kv, w)  # (slots outside the cache: nothing is appended)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(x, res, pos, slots, cu, kv, w)
    audio = torch.empty(B, d.hop * T, device="cuda")
    for step in range(3):
        n = [lens[b] + step for b in range(B)]
        x.copy_(randn(50 + step, B, C, dtype=bf))
        res.copy_(randn(60 + step, B, C, dtype=bf))
        pos.copy_(torch.tensor(n))
        slots.copy_(torch.tensor([slot_of(b, n[b]) for b in range(B)]))
        kv.copy_(torch.tensor([v + 1 for v in n]))
        g.replay()
        d.decode_device(w["z"], audio)
        d.sync()
        torch.cuda.synchronize()
        check(pos, [0, 1], w)
        want = d.decode(w["z"].view(B, 64, T).cpu().numpy())
        assert np.array_equal(audio.cpu().numpy(), want)
    d.close()
