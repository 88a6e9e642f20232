"""Edges of the decoder-layer operators (spinnv2_b200.transformer): values that are not finite or lie at the
ends of their types, empty dimensions, sizes past 32 bits, other streams."""

from __future__ import annotations

import math

import pytest
import torch

from test_transformer import F32, TYPES, U, attention64, check_codes, codes_of, gen, inputs

gpu_test = pytest.mark.gpu


# ------------------------------------------------------------------ attention
@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,hq,hk,d", [(40, 4, 4, 64), (40, 8, 2, 128), (50, 6, 2, 64), (130, 3, 1, 104), (1, 4, 2, 64),
                                        (5, 10, 2, 128), (33, 2, 2, 200)])
def test_query_that_is_not_finite_stays_alone(gpu, lq, hq, hk, d, dtype):
    """A row of queries that holds an infinity or a NaN changes no other row, bit by bit, also where an entry's
    keys are fewer than the parts that they are divided into; and a row without keys is 0 whatever it holds."""
    from spinnv2_b200 import transformer as T

    for keys in (520, 2100):
        lengths = torch.tensor([0, 1, 100, 300, keys, 0], dtype=torch.int32, device="cuda")
        q, k, v = inputs(len(lengths), lq, keys, hq, hk, d, dtype, 21)
        mask = torch.arange(keys, device="cuda")[None, :] < lengths[:, None]
        at = lq // 2
        for valid in ({"lengths": lengths}, {"key_mask": mask}):
            want = T.cross_attention(q, k, v, **valid)
            assert not want[lengths == 0].any()
            for bad in (math.nan, math.inf, -math.inf):
                bent = q.clone()
                bent[:, at, hq - 1] = bad
                for _ in range(3):
                    got = T.cross_attention(bent, k, v, **valid)
                    assert not got[lengths == 0].any()
                    got[:, at, hq - 1] = want[:, at, hq - 1]
                    assert torch.equal(got, want)


# ------------------------------------------------------------------ streams
@gpu_test
def test_encoder_calls_behind_queued_work(gpu):
    """An answer of the encoder holds its own images' features, also where torch's stream is still busy with
    earlier work when the next call writes the runtime's buffer, and from one current stream to another."""
    from conftest import seeded_input
    from spinnv2_b200.decoder import ImageEncoder

    first, second = (seeded_input((1, 3, 224, 224), seed=i) for i in (1, 2))
    matrix = torch.randn(8192, 8192, generator=gen(1), device="cuda")
    out = torch.empty_like(matrix)

    def busy():
        for _ in range(10):  # some 0.2 s
            torch.mm(matrix, matrix, out=out)

    busy()
    encoder = ImageEncoder("resnet50", 1)
    torch.cuda.synchronize()
    want = []
    for images in (first, second):
        want.append(encoder(images))
        torch.cuda.synchronize()
    assert not torch.equal(*want)
    busy()
    got = [encoder(first), encoder(second)]
    assert got[0].data_ptr() != encoder.features.data_ptr() and got[0].is_contiguous()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    busy()
    a = encoder(first)
    with torch.cuda.stream(torch.cuda.Stream()):
        b = encoder(second)
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    encoder.close()


# ------------------------------------------------------------------ product
@gpu_test
@pytest.mark.parametrize("activation", [None, "relu", "silu"])
@pytest.mark.parametrize("m,k,n,pitch", [(1, 64, 64, 16), (2, 2048, 200, 16), (40, 512, 1000, 16), (5000, 256, 2048, 16),
                                         (70, 333, 90, 1)])
def test_product_keeps_what_is_not_finite(gpu, m, k, n, pitch, activation):
    """A scale or bias of NaN shows in every element that it takes part in, whatever the activation, an
    infinite one in the elements that the definition makes infinite or NaN, and nowhere else.  The sizes
    reach one CTA a tile, clusters, pairs and the CUDA-core kernel."""
    from spinnv2_b200 import transformer as T

    g = gen(m + n)
    a, w = codes_of(m, k, g, pitch), codes_of(n, k, g, pitch)
    sa = torch.rand(m, generator=g, device="cuda") + 0.1
    sw = (torch.rand(n, generator=g, device="cuda") + 0.1) / (5000 * math.sqrt(k))
    bias = torch.randn(n, generator=g, device="cuda")
    clean = {t: T.linear_i8(a, sa, w, sw, bias=bias, activation=activation, dtype=t) for t in TYPES}
    rows, columns = torch.zeros(m, dtype=torch.bool, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
    rows[m // 2], columns[[0, n - 1, n // 3]] = True, True
    sa[m // 2], sw[0], bias[n - 1], bias[n // 3] = math.nan, math.nan, math.nan, math.inf
    v = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double() + bias.double()
    want = torch.relu(v) if activation == "relu" else v * torch.sigmoid(v) if activation == "silu" else v
    for dtype in TYPES:
        got = T.linear_i8(a, sa, w, sw, bias=bias, activation=activation, dtype=dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        keep = ~(rows[:, None] | columns)
        assert torch.equal(got[keep], clean[dtype][keep])
    bias[n // 3] = -math.inf
    if activation == "relu":
        got = T.linear_i8(a, sa, w, sw, bias=bias, activation=activation, dtype=torch.float32)
        keep = torch.ones(m, dtype=torch.bool, device="cuda")
        keep[m // 2] = False
        assert not got[keep, n // 3].any()


@gpu_test
def test_check_waits_for_every_stream(gpu):
    """check() answers for all calls before it, on whatever stream."""
    from spinnv2_b200 import transformer as T

    side = torch.cuda.Stream()
    matrix = torch.randn(8192, 8192, generator=gen(1), device="cuda")
    q, k, v = inputs(2, 40, 300, 4, 2, 64, torch.bfloat16)
    out, answer = torch.empty_like(matrix), torch.empty_like(q)
    torch.mm(matrix, matrix, out=out)  # loaded: a first launch may wait for the device
    T.cross_attention(q, k, v, out=answer)
    T.check()
    with torch.cuda.stream(side):
        for _ in range(10):  # some 0.2 s
            torch.mm(matrix, matrix, out=out)
    T.cross_attention(q, k, v, out=answer, stream=side)
    assert not side.query()
    T.check()
    assert side.query()


# ------------------------------------------------------------------ empty dimensions
@gpu_test
@pytest.mark.parametrize("shape", [(2, 0), (0, 2), (0, 0), (3, 0, 2), (0,), (2, 5, 0)])
def test_nothing_to_write(gpu, shape):
    """A call with an empty dimension, wherever it is, answers with an empty tensor of its shape."""
    from spinnv2_b200 import transformer as T

    for dtype in TYPES:
        x = torch.zeros(*shape, 64, dtype=dtype, device="cuda")
        w = torch.ones(64, dtype=dtype, device="cuda")
        for residual in (None, x.clone()):
            codes, scale, total = T.rms_norm_i8(x, w, residual)
            assert codes.shape == total.shape == x.shape and scale.shape == shape and total.dtype is dtype
        codes, scale = T.quantize_rows_i8(x)
        assert codes.shape == x.shape and scale.shape == shape
        assert T.dequantize_rows_i8(codes, scale, dtype).shape == x.shape
        weight, ws = torch.zeros(48, 64, dtype=torch.int8, device="cuda"), torch.ones(48, device="cuda")
        y = T.linear_i8(codes, scale, weight, ws, activation="relu", dtype=dtype)
        assert y.shape == (*shape, 48) and y.dtype is dtype
    given = torch.zeros(*shape, 64, dtype=torch.int8, device="cuda")
    assert T.quantize_rows_i8(x, out=given)[0] is given


@gpu_test
def test_layer_of_no_tokens(gpu):
    from spinnv2_b200.decoder import CrossAttentionLayer

    layer = CrossAttentionLayer.random(256, 128, 4, 2, 64)
    states = layer.states(torch.randn(2, 9, 128, device="cuda"))
    x = torch.zeros(2, 0, 256, dtype=torch.bfloat16, device="cuda")
    y, stream = layer.step(x, x.clone(), states)
    assert y.shape == stream.shape == x.shape
    y, _ = layer.step(x[:0], None, [t[:0] for t in states])
    assert y.shape == (0, 0, 256)
    none = layer.states(torch.zeros(2, 0, 128, device="cuda"))  # images of no positions
    y, _ = layer.step(torch.ones(2, 3, 256, dtype=torch.bfloat16, device="cuda"), None, none)
    assert y.shape == (2, 3, 256) and not y.any()


@gpu_test
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_values_of_very_many_rows(gpu, dtype):
    """As many rows as an extent can have, of one code each: more pieces than 32 bits count."""
    from spinnv2_b200 import transformer as T

    rows = 2**30 + 11
    codes = torch.zeros(rows, 1, dtype=torch.int8, device="cuda")
    scale = torch.full((rows,), 0.5, device="cuda")
    ends = [slice(0, 1000), slice(2**29 - 500, 2**29 + 500), slice(rows - 1000, rows)]
    for i, at in enumerate(ends):
        codes[at, 0] = torch.randint(-127, 128, (1000,), generator=gen(i), device="cuda").to(torch.int8)
    got = T.dequantize_rows_i8(codes, scale, dtype)
    for at in ends:
        assert torch.equal(got[at], (codes[at].float() * 0.5).to(dtype))
    assert int(torch.count_nonzero(got)) == int(torch.count_nonzero(codes))


# ------------------------------------------------------------------ norm and codes
# Widths: a unit of 16 bytes, rows that share a warp, rows of two warps that share a block, rows of many warps,
# rows read twice; each also where rows do not lie on 16-byte boundaries.
@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [3, 8, 64, 100, 250, 1000, 1024, 2048, 5001, 16384, 40000])
def test_norm_of_rows_of_any_size(gpu, width, dtype):
    """The scale of every finite row is what the definition gives, also where the squares of its values leave
    fp32's range, or their products with the weights do.  The products are formed after the row was scaled by a
    power of two, so the bounds are those of ordinary rows."""
    from spinnv2_b200 import transformer as T

    info = torch.finfo(dtype)
    g = gen(width)
    x = torch.randn(14, width, generator=g, device="cuda", dtype=torch.float64)
    low = info.smallest_normal * 2.0**-8 if dtype is not torch.float32 else info.smallest_normal
    sizes = [1.0, info.max / 64, 1e4, info.max / 2**40, info.max**0.5, info.tiny**0.5, 2**-12, low * 64, info.tiny * 2**30, 0.0]
    for i, size in enumerate(sizes):
        x[i] *= min(size, info.max / 64)
    x[10] = 0
    x[10, width - 1] = info.smallest_normal  # one small value
    x[11, width // 2] = info.max  # one huge value beside ordinary ones
    x[12] *= info.tiny
    x[12, 0] = 1.0  # one ordinary value beside tiny ones
    x[13] = info.max
    x = x.to(dtype)
    assert torch.isfinite(x).all()
    r = (0.5 * torch.randn(x.shape, generator=g, device="cuda").double() * x.double()).to(dtype)
    r = torch.where(torch.isfinite(x.float() + r.float()), r, 0)
    ordinary = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(dtype)
    wide = ordinary.clone()
    if width > 3 and dtype is not torch.float16:
        wide[1], wide[2] = 1e30, 1e-30
    for weight in (ordinary, wide):
        for eps in (0.0, 1e-6):
            for residual in (None, r):
                s = x.double() if residual is None else (x.float() + residual.float()).double()
                mean = s.square().mean(-1, keepdim=True) + eps
                y = torch.where(mean > 0, s * weight.double() / mean.sqrt(), 0.0)
                top = y.abs().amax(-1)
                assert torch.isfinite(top).all() and float(top.max()) < 1e38
                codes, scale, _ = T.rms_norm_i8(x, weight, residual, eps=eps)
                check_codes(codes, scale, y, width)
                far = torch.zeros(14, width + 1, dtype=dtype, device="cuda")[:, 1:]  # rows off their boundaries
                far.copy_(x)
                again = T.rms_norm_i8(far, weight, residual, eps=eps)
                assert torch.equal(again[0], codes) and torch.equal(again[1], scale)


@gpu_test
@pytest.mark.parametrize("b,lq,lk,hq,hk,d", [(1, 1, 200, 2, 2, 64), (2, 5, 70, 4, 2, 32), (1, 40, 300, 4, 2, 128),
                                             (8, 130, 130, 16, 16, 40), (1, 33, 1500, 2, 1, 64), (2, 3, 40, 2, 2, 7)])
def test_fp32_attention_with_values_at_the_end_of_the_type(gpu, b, lq, lk, hq, hk, d):
    """Infinities and values next to the largest one, in keys and values that count: an answer is infinite, NaN
    or finite as the definition says."""
    from spinnv2_b200 import transformer as T

    q, k, v = inputs(b, lq, lk, hq, hk, d, torch.float32, 31)
    q, k = q * 0.2, k * 0.2  # no probability underflows
    big = torch.finfo(torch.float32).max
    group = hq // hk
    for junk in (math.inf, -math.inf, big, -big):
        vv = v.clone()
        vv[0, lk // 2, hk - 1, d - 1] = junk
        got = T.cross_attention(q, k, vv)
        want, size, score = attention64(q, k, vv, None, 1 / math.sqrt(d))
        clean = T.cross_attention(q, k, v)
        other = torch.ones_like(got, dtype=torch.bool)
        other[0, :, hq - group:] = False
        assert torch.equal(got[other], clean[other])  # of other entries and heads
        if math.isinf(junk):
            hit = torch.zeros_like(other)
            hit[0, :, hq - group:, d - 1] = True
            assert (got[hit] == junk).all()
            want, size, _ = attention64(q, k, v, None, 1 / math.sqrt(d))
            got = torch.where(hit, want.float(), got)
        tol = (lk + 64) * 8 * F32 * size + 2 * ((d + 16) * 4 * F32 * score + 64 * F32) * size
        assert ((got.double() - want).abs() <= tol).all()
    # A key of -infinity where the query is positive has no weight; one of +infinity leaves no number.
    q[..., 0] = q[..., 0].abs() + 0.1
    clean = T.cross_attention(q, k, v)
    other = torch.ones_like(clean, dtype=torch.bool)
    other[0, :, :group] = False
    valid = torch.ones(b, lk, dtype=torch.bool, device="cuda")
    valid[0, lk // 3] = False
    want, size, score = (t[0, :, :group] for t in attention64(q, k, v, valid, 1 / math.sqrt(d)))
    for junk in (math.inf, -math.inf):
        kk = k.clone()
        kk[0, lk // 3, 0, 0] = junk
        got = T.cross_attention(q, kk, v)
        assert torch.equal(got[other], clean[other])
        got = got[0, :, :group]
        if junk > 0:
            assert torch.isnan(got).all()
        else:
            tol = (lk + 64) * 8 * F32 * size + 2 * ((d + 16) * 4 * F32 * score + 64 * F32) * size
            assert ((got.double() - want).abs() <= tol).all()


# ------------------------------------------------------------------ build
def test_binding_is_built_for_the_torch_that_is_there(built, monkeypatch, tmp_path):
    """The binding is compiled again for another torch or interpreter, and not otherwise."""
    from spinnv2_b200.csrc import build as b

    calls = []

    def compiler(cmd, **_):
        calls.append(cmd)
        (tmp_path / "ops.so").write_text("")
        return b.subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b, "BINDING_PATH", tmp_path / "ops.so")
    monkeypatch.setattr(b, "BINDING_STAMP", tmp_path / "ops.for")
    monkeypatch.setattr(b.subprocess, "run", compiler)
    for _ in range(2):
        assert b.build_binding() == tmp_path / "ops.so" and len(calls) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    b.build_binding()
    assert len(calls) == 2
    b.build_binding()
    assert len(calls) == 2
    monkeypatch.setattr(b.sys.implementation, "cache_tag", "cpython-1")
    b.build_binding()
    assert len(calls) == 3


def test_build_without_torch(built, monkeypatch, capsys):
    """build() compiles the graph runtime where torch is not installed, and says what it left out."""
    import sys

    import __graft_entry__

    monkeypatch.setitem(sys.modules, "torch", None)
    __graft_entry__.build()
    assert "torch is not installed" in capsys.readouterr().out


# ------------------------------------------------------------------ sizes past 32 bits, threads
@gpu_test
def test_product_of_more_than_2_to_31_answers(gpu):
    from spinnv2_b200 import transformer as T

    m, k, n = 70001, 64, 32768
    g = gen(3)
    a, w = codes_of(m, k, g), codes_of(n, k, g)
    sa, sw = torch.rand(m, generator=g, device="cuda") + 0.1, torch.rand(n, generator=g, device="cuda") / 10000
    y = T.linear_i8(a, sa, w, sw)
    for at in (slice(0, 200), slice(65436, 65636), slice(m - 200, m)):  # 2^31 answers end at row 65536
        exact = (a[at].double() @ w.double().t()) * sa[at, None].double() * sw.double()
        assert ((y[at].double() - exact).abs() <= (U[y.dtype] + 4 * F32) * exact.abs()).all()


@gpu_test
@pytest.mark.parametrize("offset", [0, 1])
def test_rows_of_more_than_2_to_31_values(gpu, offset):
    from spinnv2_b200 import transformer as T

    rows, width = 2**19 + 137, 4096
    ends = [slice(0, 50), slice(2**19 - 25, 2**19 + 25), slice(rows - 50, rows)]  # 2^31 values end at row 2^19
    flat = torch.zeros(rows * width + offset, dtype=torch.bfloat16, device="cuda")
    x = flat[offset:].view(rows, width)
    w = (1 + 0.2 * torch.randn(width, generator=gen(1), device="cuda")).bfloat16()
    for i, at in enumerate(ends):
        x[at] = torch.randn(50, width, generator=gen(i + 2), device="cuda").bfloat16()
    keep = [x[at].clone() for at in ends]
    codes, scale, total = T.rms_norm_i8(x, w, x, sum_out=x)
    assert total is x
    values = T.dequantize_rows_i8(codes, scale)
    for at, part in zip(ends, keep):
        s = 2 * part.double()
        y = s * w.double() / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        check_codes(codes[at], scale[at], y, width)
        assert torch.equal(x[at], 2 * part)
        assert torch.equal(values[at], (codes[at].float() * scale[at, None]).bfloat16())
    assert int(torch.count_nonzero(scale)) == 150


@gpu_test
def test_calls_from_two_threads(gpu):
    """Calls from two threads, each on a stream of its own, answer as they do one after another."""
    from concurrent.futures import ThreadPoolExecutor

    from spinnv2_b200 import transformer as T

    def call(seed):
        x = torch.randn(60, 1024, generator=gen(seed), device="cuda").bfloat16()
        weight = torch.randint(-127, 128, (512, 1024), generator=gen(seed + 1), device="cuda", dtype=torch.int8)
        codes, scale, _ = T.rms_norm_i8(x, x[0].contiguous())
        q = T.linear_i8(codes, scale, weight, scale.new_full((512,), 1e-3)).view(2, 30, 8, 64)
        return T.cross_attention(q, q[:, :, :4], q[:, :, 4:])

    def many(seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [call(seed) for _ in range(200)]
            torch.cuda.current_stream().synchronize()
            return got

    want = [call(seed) for seed in (1, 50)]
    with ThreadPoolExecutor(2) as pool:
        for got, one in zip(pool.map(many, (1, 50)), want):
            assert all(torch.equal(t, one) for t in got)
    T.check()


# ------------------------------------------------------------------ refusals
def test_answers_in_one_place_are_refused(built):
    """A stride of 0 between answers is a bad argument, before any CUDA call; of a dimension of one it is none."""
    from test_transformer import CROSS, c_function

    fake = 4096  # never read
    base = dict(q=fake, k=fake, v=fake, o=fake, l=0, m=0, b=2, lq=3, lk=1)
    base.update({f"st{i}": 8 for i in range(12)}, ms=0, h=2, hk=1, d=300, t=1, sc=1.0, r=0)  # too wide: no launch
    for i in (9, 10, 11):
        assert c_function("spkv2_cuda_cross_attention")(CROSS.pack(*{**base, f"st{i}": 0}.values()), None) == -1
        one = {**base, f"st{i}": 0, "b": 1, "lq": 1, "h": 1}
        assert c_function("spkv2_cuda_cross_attention")(CROSS.pack(*one.values()), None) == -43
    for i in range(9):  # inputs may
        assert c_function("spkv2_cuda_cross_attention")(CROSS.pack(*{**base, f"st{i}": 0}.values()), None) == -43
