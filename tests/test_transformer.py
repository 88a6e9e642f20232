"""The INT8 decoder-layer operators (spinnv2_b200.transformer) against their definitions in 64 bits.

Tolerances follow from the arithmetic.  u is the unit roundoff of the output type; fp32 work contributes a
few multiples of 2^-24 per operation, summed sizes included.
"""

from __future__ import annotations

import ctypes
import math
import struct
import subprocess
from pathlib import Path

import pytest
import torch

F32 = 2.0**-24
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu_test = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def close(got, want, tol):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {((got - want).abs() - tol).max().item():.3g} over"


# ------------------------------------------------------------------ norm and codes
def check_codes(codes, scale, y, width):
    """Codes and scales of the 64-bit values y.  The sum of squares adds width terms, pairwise beyond a
    thread's own, which moves the scale by width / 256 roundings at most; a code's own value is a product
    of four fp32 factors of up to 127."""
    top = y.abs().amax(dim=-1)
    close(scale, top / 127, (width / 256 + 24) * F32 * top / 127 + TINY[torch.float32])
    safe = torch.where(top > 0, top, 1.0)[..., None]
    exact = y * 127 / safe
    close(codes, exact, 0.5 + 127 * 8 * F32)
    assert int(codes.min()) >= -127


WIDTHS = [1, 2, 7, 8, 31, 64, 100, 128, 255, 256, 1000, 1024, 2047, 2048, 4096, 5000, 8192, 8200, 16384, 40000]


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_rms_norm(gpu, width, dtype):
    from spinnv2_b200 import transformer as T

    for rows in (1, 3, 67):
        for residual in (False, True):
            g = gen(width + rows)
            x = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
            r = torch.randn(rows, width, generator=g, device="cuda").to(dtype) if residual else None
            w = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(dtype)
            codes, scale, total = T.rms_norm_i8(x, w, r, eps=1e-5)
            s = x.double() + (r.double() if residual else 0)
            y = s * w.double() / (s.square().mean(-1, keepdim=True) + 1e-5).sqrt()
            check_codes(codes, scale, y, width)
            if residual:
                assert torch.equal(total, (x.float() + r.float()).to(dtype))
            else:
                assert total is x


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize_and_back(gpu, width, dtype):
    from spinnv2_b200 import transformer as T

    for rows in (1, 5, 300):
        x = (3 * torch.randn(rows, width, generator=gen(width), device="cuda")).to(dtype)
        codes, scale = T.quantize_rows_i8(x)
        assert codes.stride(0) % 16 == 0 or rows == 1
        check_codes(codes, scale, x.double(), width)
        for out in TYPES:
            y = T.dequantize_rows_i8(codes, scale, out)
            assert torch.equal(y, (codes.float() * scale[:, None]).to(out))


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [8, 100, 4096, 40000])
def test_rows_in_place_and_strided(gpu, width, dtype):
    from spinnv2_b200 import transformer as T

    g = gen(5)
    w = torch.ones(width, dtype=dtype, device="cuda")
    buf = torch.randn(9, 3, width + 3, generator=g, device="cuda").to(dtype)
    for view in (buf[:, 1, :width], buf[:, 1, 3:], buf[::2, 0, 1 : width + 1]):
        x = view.clone()
        r = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        want = T.rms_norm_i8(x, w, r)
        got = T.rms_norm_i8(view, w, r)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        codes = torch.zeros(x.shape[0], width + 5, dtype=torch.int8, device="cuda")[:, 3 : 3 + width]
        keep = r.clone()
        a = T.rms_norm_i8(view, w, keep, sum_out=keep, out=codes)  # the residual stream in place
        assert torch.equal(keep, want[2]) and torch.equal(codes, want[0]) and torch.equal(a[1], want[1])
        b = T.rms_norm_i8(x, w, r, sum_out=x)
        assert torch.equal(x, want[2]) and torch.equal(b[0], want[0])
    one = buf[:1, 0, :width].expand(4, width)  # one row for all
    codes, scale = T.quantize_rows_i8(one)
    first = T.quantize_rows_i8(one[:1].clone())
    assert torch.equal(codes, first[0].expand(4, width)) and torch.equal(scale, first[1].expand(4))


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [3, 64, 2048, 40000])
def test_rows_of_zeros_and_not_finite(gpu, width, dtype):
    from spinnv2_b200 import transformer as T

    x = torch.randn(8, width, generator=gen(1), device="cuda").to(dtype)
    x[1] = 0
    x[2, width - 1] = math.inf
    x[3, 0] = math.nan
    x[4, width // 2] = -math.inf
    tiny = TINY[dtype] if dtype is not torch.float32 else 2.0**-140
    x[5] = 0
    x[5, width - 1] = tiny  # a denormal row: its maximum is code 127
    big = torch.finfo(dtype).max
    x[6, 0] = -big
    w = torch.ones(width, dtype=dtype, device="cuda")
    for codes, scale in (T.quantize_rows_i8(x), T.rms_norm_i8(x, w, eps=0.0)[:2]):
        assert int(codes[1].abs().max()) == 0 and float(scale[1]) == 0.0
        for i in (2, 3, 4):
            assert math.isnan(float(scale[i])) and int(codes[i].abs().max()) == 0
        assert int(codes[0].abs().max()) == 127 and int(codes[7].abs().max()) == 127
        assert int(codes[5, width - 1]) == 127 and int(codes[6, 0]) == -127
    assert math.isfinite(float(T.quantize_rows_i8(x)[1][6]))


@gpu_test
def test_rows_other_ranks_and_none(gpu):
    from spinnv2_b200 import transformer as T

    x = torch.randn(2, 3, 5, 64, generator=gen(2), device="cuda")
    w = torch.ones(64, device="cuda")
    flat = T.rms_norm_i8(x.reshape(-1, 64), w)
    got = T.rms_norm_i8(x, w)
    assert got[0].shape == x.shape and got[1].shape == x.shape[:-1]
    assert torch.equal(got[0].reshape(-1, 64), flat[0]) and torch.equal(got[1].reshape(-1), flat[1])
    line = T.quantize_rows_i8(x[0, 0, 0])
    assert torch.equal(line[0], T.quantize_rows_i8(x)[0][0, 0, 0]) and line[1].shape == ()
    none = T.rms_norm_i8(x[:0], w)
    assert none[0].shape == (0, 3, 5, 64) and none[1].shape == (0, 3, 5)
    assert T.dequantize_rows_i8(none[0], none[1]).shape == (0, 3, 5, 64)
    with pytest.raises(ValueError):
        T.rms_norm_i8(x.transpose(0, 1), w)


# ------------------------------------------------------------------ product
def codes_of(rows, width, g, pitch=16):
    full = torch.randint(-128, 128, (rows, (width + pitch - 1) // pitch * pitch), generator=g, device="cuda",
                         dtype=torch.int8)
    return full[:, :width]


def check_linear(y, a, sa, w, sw, bias, act):
    acc = a.double() @ w.double().t()  # exact: below 2^53
    prod = acc * sa.double()[:, None] * sw.double()[None, :]
    v = prod if bias is None else prod + bias.double()[None, :]
    tol = 3 * F32 * (prod.abs() + (0 if bias is None else bias.double().abs()[None, :]))
    if act == "relu":
        v = v.clamp(min=0)
    elif act == "silu":
        v = v * torch.sigmoid(v)
        tol = 1.2 * tol + 16 * F32 * v.abs()
    u = U[y.dtype]
    close(y, v, tol * (1 + u) + u * v.abs() + TINY[y.dtype])


LINEAR = [(1, 1, 1), (1, 16, 8), (1, 64, 64), (2, 2048, 100), (3, 1000, 1000), (7, 129, 257), (8, 4096, 128),
          (16, 512, 1024), (17, 520, 300), (32, 2048, 2048), (33, 96, 513), (64, 384, 640), (65, 128, 128),
          (127, 2000, 255), (128, 128, 256), (129, 640, 1030), (255, 1024, 96), (300, 777, 771), (513, 256, 4100),
          (1000, 2048, 1000), (4099, 320, 131)]


@gpu_test
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear(gpu, m, k, n):
    from spinnv2_b200 import transformer as T

    g = gen(m * 7 + k * 3 + n)
    a, w = codes_of(m, k, g), codes_of(n, k, g)
    sa = torch.rand(m, generator=g, device="cuda") + 0.1
    sw = (torch.rand(n, generator=g, device="cuda") + 0.1) / (5000 * math.sqrt(k))
    bias = torch.randn(n, generator=g, device="cuda")
    for dtype in TYPES:
        for b, act in ((None, None), (bias, "relu"), (bias, "silu")):
            y = T.linear_i8(a, sa, w, sw, bias=b, activation=act, dtype=dtype)
            check_linear(y, a, sa, w, sw, b, act)
            assert torch.equal(y, T.linear_i8(a, sa, w, sw, bias=b, activation=act, dtype=dtype))


@gpu_test
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_linear_strides_and_alignment(gpu, m):
    from spinnv2_b200 import transformer as T

    g = gen(m)
    k, n = 333, 210
    sa, sw = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda") / 10000
    a0, w0 = codes_of(m, k, g), codes_of(n, k, g)
    want = T.linear_i8(a0, sa, w0, sw, dtype=torch.float32)
    check_linear(want, a0, sa, w0, sw, None, None)
    packed_a, packed_w = a0.clone(memory_format=torch.contiguous_format), w0.contiguous()  # rows 333 bytes apart
    odd_a = torch.empty(m, k + 14, dtype=torch.int8, device="cuda")[:, 3 : 3 + k].copy_(a0)
    odd_w = torch.empty(n * k + 5, dtype=torch.int8, device="cuda")[5:].view(n, k).copy_(w0)
    wide = torch.empty(m, 3, n + 1, device="cuda")
    for a in (a0, packed_a, odd_a):
        for w in (w0, packed_w, odd_w):
            assert torch.equal(T.linear_i8(a, sa, w, sw, dtype=torch.float32), want)
            out = wide[:, 1, 1:]
            assert T.linear_i8(a, sa, w, sw, out=out) is out and torch.equal(out, want)
    for dtype in (torch.float16, torch.bfloat16):
        out = torch.zeros(m, n + 2, dtype=dtype, device="cuda")
        T.linear_i8(a0, sa, w0, sw, out=out[:, 1 : n + 1])
        assert torch.equal(out[:, 1 : n + 1], want.to(dtype)) and not out[:, 0].any() and not out[:, -1].any()
    row = a0[:1].expand(m, k)
    assert torch.equal(T.linear_i8(row, sa, w0, sw, dtype=torch.float32),
                       T.linear_i8(row.contiguous(), sa, w0, sw, dtype=torch.float32))


@gpu_test
def test_linear_extremes(gpu):
    from spinnv2_b200 import transformer as T

    k = 131071  # the largest k: 128 * 128 * k is the largest sum that int32 holds
    for m in (1, 130):
        a = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
        w = torch.full((130, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
        w[1] = 127
        one = torch.ones(130, device="cuda")
        y = T.linear_i8(a, one[:m], w, one, dtype=torch.float32)
        assert float(y[0, 0]) == float(torch.tensor(float(128 * 128 * k), dtype=torch.float32))
        assert float(y[m - 1, 1]) == float(torch.tensor(float(-128 * 127 * k), dtype=torch.float32))
    empty = T.linear_i8(a[:, :0], one[:1].expand(130).contiguous(), w[:, :0], one, bias=one, dtype=torch.float32)
    assert torch.equal(empty, torch.ones(130, 130, device="cuda"))
    assert T.linear_i8(a[:0], one[:0], w, one).shape == (0, 130)
    assert T.linear_i8(a, torch.ones(130, device="cuda"), w[:0], one[:0]).shape == (130, 0)
    nan = torch.full((130,), math.nan, device="cuda")  # the scale of a row that was not finite
    assert torch.isnan(T.linear_i8(a, nan, w, one)).all()
    x = torch.randint(-128, 128, (2, 3, 64), device="cuda", dtype=torch.int8)
    s = torch.rand(2, 3, device="cuda")
    ww, sw = torch.randint(-128, 128, (48, 64), device="cuda", dtype=torch.int8), torch.rand(48, device="cuda")
    y = T.linear_i8(x, s, ww, sw)
    assert y.shape == (2, 3, 48)
    assert torch.equal(y.reshape(6, 48), T.linear_i8(x.reshape(6, 64), s.reshape(6), ww, sw))


# ------------------------------------------------------------------ attention
def attention64(q, k, v, valid, scale):
    """(answer, sum of p |v|, largest sum of |q k| scale) in 64 bits; zeros for a row without keys."""
    b, lq, hq, d = q.shape
    hk = k.shape[2]
    group = hq // hk
    q, k, v = (t.double() for t in (q, k, v))
    if valid is not None:
        k = torch.where(valid[:, :, None, None], k, 0.0)
        v = torch.where(valid[:, :, None, None], v, 0.0)
    k, v = (t.repeat_interleave(group, dim=2) for t in (k, v))
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) * scale
    size = torch.einsum("bqhd,bkhd->bhqk", q.abs(), k.abs()) * abs(scale)
    if valid is not None:
        s = s.masked_fill(~valid[:, None, None, :], -math.inf)
    if s.shape[-1] == 0:
        zero = torch.zeros_like(q)
        return zero, zero, torch.zeros(b, lq, hq, 1, device=q.device, dtype=torch.float64)
    p = torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0)
    o = torch.einsum("bhqk,bkhd->bqhd", p, v)
    a = torch.einsum("bhqk,bkhd->bqhd", p, v.abs())
    return o, a, size.amax(dim=-1).transpose(1, 2)[..., None]


def check_attention(out, q, k, v, valid, scale):
    """A score sums width products, in an order and with roundings of the kernel's choice (2^-22 each, of the
    sum of the terms' sizes); that error, twice (numerator and denominator), moves a probability by as much.
    In 16-bit types each probability is rounded once before it meets its value, and the answer once more."""
    o, a, size = attention64(q, k, v, valid, scale)
    u = U[q.dtype]
    score = (q.shape[3] + 16) * 4 * F32 * size + 64 * F32
    close(out, o, u * (o.abs() + a) + 2 * score * a + (k.shape[1] + 64) * 4 * F32 * a + TINY[q.dtype])


def inputs(b, lq, lk, hq, hk, d, dtype, seed=0):
    g = gen(seed)
    q = (1.5 * torch.randn(b, lq, hq, d, generator=g, device="cuda")).to(dtype)
    kv = torch.randn(b, lk, 2, hk, d, generator=g, device="cuda").to(dtype)
    return q, kv[:, :, 0], kv[:, :, 1]


SHAPES = [  # batch, queries, keys, heads, kv_heads, width
    (1, 1, 1, 1, 1, 64), (1, 1, 49, 16, 16, 64), (3, 1, 130, 8, 2, 128), (2, 1, 1000, 4, 4, 80), (1, 1, 4097, 8, 1, 128),
    (2, 3, 63, 6, 2, 64), (2, 4, 64, 4, 1, 40), (5, 1, 65, 32, 4, 96), (2, 16, 127, 2, 2, 128), (1, 17, 129, 4, 2, 64),
    (1, 2, 300, 64, 2, 32), (2, 64, 128, 3, 3, 64), (1, 65, 257, 4, 4, 128), (1, 100, 850, 8, 8, 32), (2, 77, 196, 12, 12, 64),
    (1, 128, 1, 2, 2, 64), (1, 129, 384, 2, 1, 128), (2, 300, 200, 4, 2, 64), (1, 257, 1025, 8, 2, 128), (1, 31, 33, 5, 5, 7),
    (1, 40, 70, 2, 2, 130), (2, 1, 90, 4, 2, 256), (1, 33, 129, 2, 1, 200), (1, 600, 513, 3, 3, 96), (1, 1, 20000, 2, 2, 64),
    (70, 1, 3, 2, 1, 16), (1, 130, 129, 2, 2, 8), (3, 5, 0, 2, 2, 64),
    (20, 400, 300, 4, 4, 128), (10, 130, 129, 32, 8, 96), (40, 450, 64, 2, 2, 128), (19, 513, 640, 4, 4, 104)]


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(gpu, shape, dtype):
    from spinnv2_b200 import transformer as T

    b, lq, lk, hq, hk, d = shape
    q, k, v = inputs(*shape, dtype)
    out = T.cross_attention(q, k, v)
    check_attention(out, q, k, v, None, 1 / math.sqrt(d))
    assert torch.equal(out, T.cross_attention(q, k, v))


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_masks(gpu, shape, dtype):
    """Lengths of 0, 1, beyond the end and below 0; masks with holes; entries with nothing left.  What does
    not count is NaN, infinite or the type's lowest value."""
    from spinnv2_b200 import transformer as T

    _, lq, lk, hq, hk, d = shape
    b = 7 if lq * hq * lk < 100000 else 4
    q, k, v = inputs(b, lq, lk, hq, hk, d, dtype, 3)
    place = torch.arange(lk, device="cuda")[None, :]
    lengths = torch.tensor([0, 1, lk + 9, lk // 2, -4, max(lk - 1, 0), 64][-b:], dtype=torch.int32, device="cuda")
    by_length = place < lengths[:, None]
    holes = torch.rand(b, lk, generator=gen(4), device="cuda") < 0.6
    holes[1] = False
    if lk:
        holes[2] = place[0] == lk - 1
        holes[3, : lk // 2] = False
    for use_l, use_m in ((True, False), (False, True), (True, True)):
        valid = torch.ones(b, lk, dtype=torch.bool, device="cuda")
        valid &= by_length if use_l else True
        valid &= holes if use_m else True
        kk, vv = k.clone(), v.clone()
        for n, junk in enumerate((math.nan, math.inf, torch.finfo(dtype).min)):
            off = ~valid & (place % 3 == n)
            kk[off] = junk
            vv[off] = junk
        out = T.cross_attention(q, kk, vv, lengths=lengths if use_l else None, key_mask=holes if use_m else None)
        check_attention(out, q, kk, vv, valid, 1 / math.sqrt(d))
        assert not out[~valid.any(dim=1)].any()


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,hq,hk", [(1, 8, 2), (5, 4, 4), (150, 4, 2)])
def test_attention_strides(gpu, dtype, lq, hq, hk):
    from spinnv2_b200 import transformer as T

    b, lk, d = 3, 150, 64
    q, k, v = inputs(b, lq, lk, hq, hk, d, dtype, 6)
    want = T.cross_attention(q, k.contiguous(), v.contiguous())
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(T.cross_attention(*heads_first), want)
    out = torch.zeros(b, hq, lq, d, dtype=dtype, device="cuda").transpose(1, 2)
    assert T.cross_attention(q, k, v, out=out) is out and torch.equal(out, want)
    mask = torch.ones(b, 2, lk + 3, dtype=torch.uint8, device="cuda")[:, 1, 3:]  # rows apart, not aligned
    assert torch.equal(T.cross_attention(q, k, v, key_mask=mask), want)
    shared = [t[:1].expand(b, *t.shape[1:]) for t in (k, v)]  # one image for the whole batch
    got = T.cross_attention(q, *shared)
    assert torch.equal(got, T.cross_attention(q, *[t.contiguous() for t in shared]))

    def shifted(t, by):
        flat = torch.empty(t.numel() + by, dtype=dtype, device="cuda")[by:]
        return flat.view(t.shape).copy_(t)

    for by in (1, 3):
        got = T.cross_attention(shifted(q, by), shifted(k, by), shifted(v, by), out=shifted(q, by))
        check_attention(got, q, k, v, None, 1 / math.sqrt(d))


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [1, 200])
def test_attention_scores_of_any_size(gpu, dtype, lq):
    """Large scores (one key takes all), equal scores, a negative scale and scale 0, and maxima that rise from
    tile to tile."""
    from spinnv2_b200 import transformer as T

    q, k, v = inputs(2, lq, 700, 4, 2, 64, dtype, 8)
    for scale in (20.0, 1.0, 0.0, -0.5):
        check_attention(T.cross_attention(q, k, v, scale=scale), q, k, v, None, scale)
    rising = k * torch.linspace(0, 6, 700, device="cuda").to(dtype)[None, :, None, None]
    check_attention(T.cross_attention(q, rising, v), q, rising, v, None, 0.125)
    check_attention(T.cross_attention(q, rising.flip(1), v), q, rising.flip(1), v, None, 0.125)
    nan = k.clone()
    nan[0, 5, 0, 0] = math.nan  # a key that counts
    out = T.cross_attention(q, nan, v)
    assert torch.isnan(out[0, :, :2]).all() and torch.equal(out[:, :, 2:], T.cross_attention(q, k, v)[:, :, 2:])


@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [1, 100])
def test_attention_masks_that_end_early(gpu, lq, dtype):
    """Masks over many keys whose last key that counts lies anywhere: the first, the last, around the steps of
    the kernels, or nowhere; together with lengths."""
    from spinnv2_b200 import transformer as T

    ends = [0, 1, 16, 127, 128, 129, 2047, 2048, 2049, 4100, 4999, 5000]
    q, k, v = inputs(len(ends), lq, 5000, 4, 2, 64, dtype, 11)
    mask = torch.rand(len(ends), 5000, generator=gen(12), device="cuda") < 0.3
    for i, end in enumerate(ends):
        mask[i, end:] = False
        if end:
            mask[i, end - 1] = True
    off = ~mask
    k, v = k.clone(), v.clone()
    k[off] = math.nan
    v[off] = math.nan
    check_attention(T.cross_attention(q, k, v, key_mask=mask), q, k, v, mask, 0.125)
    lengths = torch.tensor([5000, 5000, 3, 5000, 100, 5000, 600, 513, 512, 511, 5000, 2500], dtype=torch.int32, device="cuda")
    both = mask & (torch.arange(5000, device="cuda")[None, :] < lengths[:, None])
    out = T.cross_attention(q, k, v, key_mask=mask, lengths=lengths)
    check_attention(out, q, k, v, both, 0.125)
    assert not out[0].any()


@gpu_test
@pytest.mark.parametrize("lq", [1, 40])
def test_attention_offsets_past_32_bits(gpu, lq):
    from spinnv2_b200 import transformer as T

    keys = 2**31 // (16 * 128) + 2000  # the last keys start beyond 2^31 elements
    k = torch.zeros(1, keys, 16, 128, dtype=torch.float16, device="cuda")
    k[:, -1500:] = torch.randn(1, 1500, 16, 128, generator=gen(1), device="cuda").half()
    q = torch.randn(1, lq, 16, 128, generator=gen(2), device="cuda").half()
    mask = torch.zeros(1, keys, dtype=torch.bool, device="cuda")
    mask[:, -70:] = True
    got = T.cross_attention(q, k, k, key_mask=mask)
    check_attention(got, q, k[:, -70:], k[:, -70:], None, 1 / math.sqrt(128))


# ------------------------------------------------------------------ streams
@gpu_test
def test_other_streams_and_capture(gpu):
    from spinnv2_b200 import transformer as T

    q, k, v = inputs(2, 3, 100, 4, 2, 64, torch.bfloat16)
    want = T.cross_attention(q, k, v)
    x = torch.randn(40, 512, generator=gen(1), device="cuda").bfloat16()
    w = torch.randint(-128, 128, (512, 512), device="cuda", dtype=torch.int8)
    ones = torch.ones(512, device="cuda")
    codes, scale = T.quantize_rows_i8(x)
    y = T.linear_i8(codes, scale, w, ones)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = T.cross_attention(q, k, v, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.stream(side):
        got = T.linear_i8(*T.quantize_rows_i8(x), w, ones)
    side.synchronize()
    assert torch.equal(got, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c2, s2 = T.quantize_rows_i8(x)
        y2 = T.linear_i8(c2, s2, w, ones)
        o2 = T.cross_attention(q, k, v)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o2, want) and torch.equal(y2, T.linear_i8(codes, scale * 2, w, ones))


# ------------------------------------------------------------------ refusals
@gpu_test
def test_refusals(gpu):
    from spinnv2_b200 import transformer as T
    from spinnv2_b200.runtime import Spkv2Error

    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for bad in (lambda: T.rms_norm_i8(x.cpu(), w), lambda: T.rms_norm_i8(x, w[:63]), lambda: T.rms_norm_i8(x, w, x[:3]),
                lambda: T.rms_norm_i8(x.t(), w[:4]), lambda: T.quantize_rows_i8(x, out=torch.zeros(4, 63, dtype=torch.int8, device="cuda")),
                lambda: T.quantize_rows_i8(x, scale_out=torch.zeros(5, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: T.rms_norm_i8(x.double(), w), lambda: T.rms_norm_i8(x, w.half()), lambda: T.quantize_rows_i8(x.int()),
                lambda: T.dequantize_rows_i8(x, w), lambda: T.rms_norm_i8(None, w)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(Spkv2Error) as e:
        T.rms_norm_i8(x, w, eps=-1.0)
    assert e.value.code == -1
    with pytest.raises(Spkv2Error):
        T.quantize_rows_i8(x, out=torch.zeros(64, dtype=torch.int8, device="cuda").expand(4, 64))

    a, b = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    s4, s8 = torch.ones(4, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: T.linear_i8(a, s8, b, s8), lambda: T.linear_i8(a, s4, b, s4), lambda: T.linear_i8(a, s4, b[:, :32], s8),
                lambda: T.linear_i8(a, s4, b, s8, bias=s4), lambda: T.linear_i8(a, s4, b, s8, activation="gelu"),
                lambda: T.linear_i8(a, s4, b, s8, out=torch.zeros(4, 9, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: T.linear_i8(x, s4, b, s8), lambda: T.linear_i8(a, s4.half(), b, s8),
                lambda: T.linear_i8(a, s4, b, s8, dtype=torch.float64)):
        with pytest.raises(TypeError):
            bad()
    long = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(Spkv2Error) as e:
        T.linear_i8(long, s4[:1], long, s4[:1])
    assert e.value.code == -43

    q, k, v = inputs(2, 3, 10, 4, 2, 64, torch.float16)
    bits = torch.ones(2, 10, dtype=torch.bool, device="cuda")
    for bad in (lambda: T.cross_attention(q[:, :, :3], k, v), lambda: T.cross_attention(q, k[:1], v[:1]),
                lambda: T.cross_attention(q, k, v[:, :9]), lambda: T.cross_attention(q[0], k, v),
                lambda: T.cross_attention(q, k, v, key_mask=bits[:, :9]), lambda: T.cross_attention(q, k[..., :32], v[..., :32]),
                lambda: T.cross_attention(q, k, v, lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: T.cross_attention(q, k, v, out=q[:, :1].expand(2, 3, 4, 64)),
                lambda: T.cross_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: T.cross_attention(q.float(), k, v), lambda: T.cross_attention(q, k, v, key_mask=bits.float()),
                lambda: T.cross_attention(q, k, v, lengths=torch.zeros(2, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(Spkv2Error) as e:
        T.cross_attention(q, k, v, scale=math.inf)
    assert e.value.code == -1
    wide = [torch.zeros(1, 1, 1, 257, device="cuda") for _ in range(3)]
    with pytest.raises(Spkv2Error) as e:
        T.cross_attention(*wide)
    assert e.value.code == -43


# The argument structs of spkv2_transformer.h, in native alignment.
NORM, CODES, LINEAR_ARGS, CROSS = (struct.Struct(f) for f in ("@6P6qfi", "@3P4qii", "@6P6qii", "@6P16q4ifi"))


def c_function(name):
    from spinnv2_b200.runtime import load_library

    fn = getattr(load_library(), name)
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
    return fn


def test_host_checks_without_a_device(built):
    """The library refuses bad arguments on the host, before any CUDA call."""

    def call(name, args):
        return c_function(name)(args, None)

    fake = 4096  # never read
    norm = lambda **c: NORM.pack(*{**dict(x=fake, r=0, w=fake, s=0, c=fake, sc=fake, rows=2, width=8, xs=8, rs=0, ss=0, cs=8, eps=0.0, t=1), **c}.values())  # noqa: E731
    for bad in (dict(x=0), dict(w=0), dict(c=0), dict(sc=0), dict(rows=-1), dict(width=0), dict(xs=-1), dict(cs=7), dict(s=fake, ss=4), dict(eps=-1.0), dict(eps=math.nan), dict(width=1 << 25),
                dict(x=fake + 2), dict(s=fake + 1, ss=8), dict(sc=fake + 2)):
        assert call("spkv2_cuda_rms_norm_i8", norm(**bad)) == -1, bad
    assert call("spkv2_cuda_rms_norm_i8", norm(t=2)) == -43
    assert call("spkv2_cuda_rms_norm_i8", norm(rows=0)) == 0
    assert c_function("spkv2_cuda_rms_norm_i8")(None, None) == -1
    lin = lambda **c: LINEAR_ARGS.pack(*{**dict(a=fake, sa=fake, w=fake, sw=fake, b=0, y=fake, m=2, n=2, k=2, as_=2, ws=2, ys=2, t=1, act=0), **c}.values())  # noqa: E731
    for bad in (dict(a=0), dict(sa=0), dict(w=0), dict(sw=0), dict(y=0), dict(m=-1), dict(k=-1), dict(as_=-1), dict(ys=1), dict(act=3), dict(act=-1),
                dict(y=fake + 2), dict(sa=fake + 1), dict(b=fake + 2)):
        assert call("spkv2_cuda_linear_i8", lin(**bad)) == -1, bad
    assert call("spkv2_cuda_linear_i8", lin(k=1 << 17)) == -43 and call("spkv2_cuda_linear_i8", lin(t=9)) == -43
    assert call("spkv2_cuda_linear_i8", lin(m=0)) == 0 and c_function("spkv2_cuda_linear_i8")(None, None) == -1
    base = dict(q=fake, k=fake, v=fake, o=fake, l=0, m=0, b=1, lq=1, lk=1)
    base.update({f"st{i}": 8 for i in range(12)}, ms=0, h=2, hk=1, d=8, t=1, sc=1.0, r=0)
    cross = lambda **c: CROSS.pack(*{**base, **c}.values())  # noqa: E731
    for bad in (dict(q=0), dict(k=0), dict(o=0), dict(b=-1), dict(lk=-1), dict(h=3, hk=2), dict(hk=0), dict(d=0), dict(st4=-1), dict(sc=math.nan), dict(m=fake, ms=-1),
                dict(q=fake + 2), dict(l=fake + 2)):
        assert call("spkv2_cuda_cross_attention", cross(**bad)) == -1, bad
    for bad in (dict(d=257), dict(t=2), dict(lk=1 << 31), dict(lq=1 << 31)):
        assert call("spkv2_cuda_cross_attention", cross(**bad)) == -43, bad
    assert call("spkv2_cuda_cross_attention", cross(lq=0)) == 0


def test_argument_layout_matches_the_header(built, tmp_path):
    """The packed arguments have the sizes of the C structs."""
    repo = Path(__file__).resolve().parents[1]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "spkv2_transformer.h"\nint main(void) { printf("%zu %zu %zu %zu %zu", '
                   "sizeof(Spkv2RmsNormI8), sizeof(Spkv2QuantizeRowsI8), sizeof(Spkv2DequantizeRowsI8), "
                   "sizeof(Spkv2LinearI8), sizeof(Spkv2CrossAttention)); return 0; }\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-I", str(repo / "include"), str(src), "-o", str(exe)], check=True)
    sizes = [int(s) for s in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [NORM.size, CODES.size, CODES.size, LINEAR_ARGS.size, CROSS.size]


def test_cpu_tensors_are_refused(built):
    from spinnv2_b200 import transformer as T

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        T.quantize_rows_i8(x)
    with pytest.raises(TypeError):
        T.quantize_rows_i8([1.0])




@gpu_test
def test_check_after_calls(gpu):
    """No wait gave up in the calls before, and the status call says so."""
    from spinnv2_b200 import transformer as T

    q, k, v = inputs(2, 40, 300, 4, 2, 64, torch.bfloat16)
    T.cross_attention(q, k, v)
    T.check()
    T.check(0)
