"""Rows in four bits: encoding and decoding equal the 64-bit definition bit for bit, products lie within the error of fp32 sums
of the 64-bit result (int4_plain.product_bound, derived there)."""
import ctypes as C

import numpy as np
import pytest

import int4_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import vectorstorekit_b200 as vsk
    d = vsk.CUDAComputeDevice(0)
    yield d
    d.close()


def _t(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _rows(rng, n, dim, kind):
    x = rng.standard_normal((n, dim))
    if kind == "shifted":
        x = x * rng.uniform(0.1, 3.0, (1, dim)) + rng.uniform(-2, 2, (1, dim))
    elif kind == "wide":      # magnitudes from 1e-4 to 1e3 in one row
        x = x * 10.0 ** rng.uniform(-4, 3, (n, dim))
    elif kind == "constant":
        x = np.repeat(rng.standard_normal((n, 1)), dim, 1)
    elif kind == "zero":
        x = np.zeros((n, dim))
    elif kind == "huge":      # scales beyond fp16
        x = x * 1e7
    elif kind == "tiny":      # scales below fp16
        x = x * 1e-9
    return x


KINDS = ["normal", "shifted", "wide", "constant", "zero", "huge", "tiny"]


@pytest.mark.parametrize("n,dim", [(1, 1), (3, 2), (5, 31), (4, 33), (7, 127), (2, 129), (33, 384), (9, 1000), (257, 70)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
def test_codec_equals_the_definition(dev, n, dim, group, symmetric):
    import torch
    import vectorstorekit_b200 as vsk
    q = vsk.Int4Quantizer(dev, group, symmetric)
    rng = np.random.default_rng(1000 * dim + group)
    for i, kind in enumerate(KINDS):
        dtype = ("f32", "f16", "bf16")[(i + dim) % 3] if kind != "huge" else "f32"
        x = torch.from_numpy(_rows(rng, n, dim, kind)).to(_t(dtype)).cuda()
        want = plain.encode(x.float().cpu().numpy(), group, symmetric)
        codes, scales, middles = q.quantizeBatch(x)
        assert np.array_equal(scales.cpu().numpy(), want[1]), kind
        assert (middles is None) == symmetric and (symmetric or np.array_equal(middles.cpu().numpy(), want[2])), kind
        assert np.array_equal(codes.cpu().numpy(), plain.pack(want[0])), kind
        exact = plain.values(*want, group).astype(np.float32)
        assert np.array_equal(q.dequantizeBatch(codes, scales, middles, dim).cpu().numpy(), exact), kind
        # host arrays: the same bytes
        hc, hs, hm = q.quantizeBatch(x.float().cpu().numpy())
        assert np.array_equal(hc, codes.cpu().numpy()) and np.array_equal(hs, want[1]) and (symmetric or np.array_equal(hm, want[2]))
        assert np.array_equal(q.dequantizeBatch(hc, hs, hm, dim), exact)


@pytest.mark.parametrize("symmetric", [True, False])
def test_codes_of_values_next_to_a_border(dev, symmetric):
    """Quotients at a half, and one fp32 step to either side of it."""
    import torch
    import vectorstorekit_b200 as vsk
    rng = np.random.default_rng(5)
    n, group = 4000, 32
    x = np.empty((n, group), np.float32)
    s = rng.uniform(0.01, 5.0, n).astype(np.float16).astype(np.float32)
    x[:, 0], x[:, 1] = 7 * s, (-7 if symmetric else -8) * s
    half = (rng.integers(-6, 6, (n, group - 2)) + 0.5).astype(np.float32) * s[:, None]
    step = rng.integers(-1, 2, half.shape)
    x[:, 2:] = np.where(step < 0, np.nextafter(half, np.float32(-1e9)), np.where(step > 0, np.nextafter(half, np.float32(1e9)), half))
    want = plain.encode(x, group, symmetric)
    codes, scales, middles = vsk.Int4Quantizer(dev, group, symmetric).quantizeBatch(torch.from_numpy(x).cuda())
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), plain.pack(want[0]))


def test_codec_leaves_the_bytes_between_rows_alone_and_takes_strided_rows(dev):
    import torch
    import vectorstorekit_b200 as vsk
    rng = np.random.default_rng(6)
    for dtype in ("f32", "f16"):
        wide = torch.from_numpy(rng.standard_normal((40, 203))).to(_t(dtype)).cuda()
        for first, dim in ((1, 101), (3, 130), (0, 200)):
            x = wide[:, first:first + dim]
            q = vsk.Int4Quantizer(dev, 32, False)
            a, b = q.quantizeBatch(x), q.quantizeBatch(x.contiguous())
            assert all(torch.equal(u, v) for u, v in zip(a, b))
        codes = torch.full((40, 77), 0xAB, dtype=torch.uint8, device="cuda")
        scales = torch.empty((40, 4), dtype=torch.float16, device="cuda")
        x = wide[:, :101].contiguous()
        torch.cuda.synchronize()
        st = dev._lib.vsk_q4_encode_dev(dev._h, C.c_void_p(x.data_ptr()), {"f32": 0, "f16": 1}[dtype], 40, 101, 101, 32, 1,
                                        C.c_void_p(codes.data_ptr()), 77, C.c_void_p(scales.data_ptr()), None) \
            if not _checked() else None
        if st is not None:
            assert st == 0
            want = plain.pack(plain.encode(x.float().cpu().numpy(), 32, True)[0])
            assert np.array_equal(codes[:, :51].cpu().numpy(), want) and bool((codes[:, 51:] == 0xAB).all())


def _checked():
    from vectorstorekit_b200 import _lib
    return _lib.CHECKED


def _case(rng, n, dim, group, symmetric):
    codes = rng.integers(0, 16, (n, dim))
    groups = -(-dim // group)
    scales = (10.0 ** rng.uniform(-3, 0, (n, groups))).astype(np.float16)
    middles = None if symmetric else rng.standard_normal((n, groups)).astype(np.float16)
    return codes, scales, middles


def _run(dev, codes, scales, middles, group, x, out, code_pad=0, scale_pad=0, x_pad=0, shift=0):
    """The product with rows that lie inside wider ones, `shift` bytes / elements behind an aligned address."""
    import torch
    import vectorstorekit_b200 as vsk
    n, width = codes.shape[0], (codes.shape[1] + 1) // 2

    def placed(a, pad, at):
        t = torch.from_numpy(a) if isinstance(a, np.ndarray) else a
        room = torch.empty(t.shape[0] * (t.shape[1] + pad) + at, dtype=t.dtype, device="cuda")
        view = room[at:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
        return view.copy_(t)

    c = placed(plain.pack(codes), code_pad, shift)
    s = placed(scales, scale_pad, shift)
    m = None if middles is None else placed(middles, scale_pad, shift)
    q = vsk.Int4Quantizer(dev, group, middles is None)
    y = q.product(placed(x, x_pad, shift), c, s, m, out_dtype=_t(out))
    assert y.shape == (x.shape[0], n) and y.dtype == _t(out) and width == c.shape[1]
    return y.float().cpu().numpy()


def _compare(got, codes, scales, middles, group, x, out):
    x64 = x.double().numpy()
    y = x64 @ plain.values(codes, scales, middles, group).T
    bound = plain.product_bound(codes, scales, middles, group, x64, y, out)
    off = np.abs(got - y)
    assert np.all(off <= bound), (float((off / bound).max()), np.argwhere(off > bound)[:4])


SHAPES = [(1, 1, 1), (1, 7, 1), (17, 33, 2), (16, 128, 1), (100, 100, 3), (257, 1000, 5), (64, 4096, 8), (33, 160, 9), (50, 129, 17),
          (40, 256, 33), (31, 384, 70), (5000, 64, 1), (3, 8192, 1), (15, 96, 2), (48, 272, 11), (1000, 768, 64), (20_001, 136, 4)]


@pytest.mark.parametrize("n,dim,nq", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
def test_products_against_64_bits(dev, n, dim, nq, group, symmetric):
    import torch
    rng = np.random.default_rng(n + 7 * dim + 13 * nq + group)
    codes, scales, middles = _case(rng, n, dim, group, symmetric)
    for kind in ("f32", "f16", "bf16"):
        x = torch.from_numpy(rng.standard_normal((nq, dim))).to(_t(kind))
        for out in {"f32", kind}:
            _compare(_run(dev, codes, scales, middles, group, x, out), codes, scales, middles, group, x, out)


@pytest.mark.parametrize("code_pad,scale_pad,x_pad,shift", [(0, 0, 0, 1), (1, 1, 1, 0), (4, 2, 8, 0), (13, 3, 5, 2), (2, 0, 0, 4), (16, 8, 16, 8)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_products_with_rows_inside_wider_ones(dev, kind, code_pad, scale_pad, x_pad, shift):
    import torch
    rng = np.random.default_rng(code_pad + 17 * shift)
    for n, dim, nq, group, symmetric in ((70, 320, 3, 32, True), (35, 1025, 10, 64, False), (18, 640, 2, 128, True)):
        codes, scales, middles = _case(rng, n, dim, group, symmetric)
        x = torch.from_numpy(rng.standard_normal((nq, dim))).to(_t(kind))
        got = _run(dev, codes, scales, middles, group, x, "f32", code_pad, scale_pad, x_pad, shift)
        _compare(got, codes, scales, middles, group, x, "f32")


# rows enough to fill the machine, at 16-byte places: one tile of 128 rows to a block and several, ends inside a tile, one step of 64 columns,
# odd numbers of steps, ends inside a group, vectors of more than one pass; and up to sixteen vectors with as many rows
@pytest.mark.parametrize("n,dim,nq", [(18_944, 64, 17), (19_073, 129, 32), (9_601, 200, 61), (40_000, 1000, 32), (152_000, 65, 40), (80_001, 321, 9),
                                      (30, 1100, 4_760)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind,symmetric", [("f16", False), ("bf16", True)])
def test_products_with_many_rows(dev, kind, symmetric, group, n, dim, nq):
    import torch
    rng = np.random.default_rng(n + dim + nq + group)
    codes, scales, middles = _case(rng, n, dim, group, symmetric)
    x = torch.from_numpy(rng.standard_normal((nq, dim))).to(_t(kind))
    width, groups = (dim + 1) // 2, scales.shape[1]
    out, scale_pad = ((kind, -groups % 4), ("f32", 1))[(n + group) // 32 % 2]
    _compare(_run(dev, codes, scales, middles, group, x, out, code_pad=-width % 16, scale_pad=scale_pad), codes, scales, middles, group, x, out)
    bad = x.clone()
    bad[nq // 2, dim - 1] = float("inf")
    got = _run(dev, codes, scales, middles, group, bad, "f32", code_pad=-width % 16)
    others = np.arange(nq) != nq // 2
    assert not np.isfinite(got[nq // 2]).any()
    assert np.array_equal(got[others], _run(dev, codes, scales, middles, group, x, "f32", code_pad=-width % 16)[others])


def test_products_of_unusual_vectors(dev):
    """fp32 values far from one, below the normal range, and with all 24 bits set; rows of one code; an fp16 result beyond its range."""
    import torch
    rng = np.random.default_rng(11)
    codes, scales, middles = _case(rng, 90, 300, 32, True)
    for size in (2.0 ** 100, 2.0 ** -100, 1.0):
        x = torch.from_numpy((rng.integers(2 ** 23, 2 ** 24, (3, 300)) * rng.choice([-1.0, 1.0], (3, 300)) * 2.0 ** -24 * size)).float()
        _compare(_run(dev, codes, scales, middles, 32, x, "f32"), codes, scales, middles, 32, x, "f32")
    ones = np.full((5, 64), 15)
    big = np.full((5, 1), 65504.0, np.float16)
    x = torch.ones((2, 64), dtype=torch.float16)
    assert np.all(np.isposinf(_run(dev, ones, big, None, 64, x, "f16")))
    assert np.all(_run(dev, ones, big, None, 64, x, "f32") == 64 * 7 * 65504.0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_products_of_vectors_with_one_element_far_above_the_others(dev, kind):
    """A thousand times the others, as activations of language models have them; rows with and without a weight at that place."""
    import torch
    rng = np.random.default_rng(13)
    codes, scales, middles = _case(rng, 80, 512, 64, True)
    codes[::2, 77] = 8
    for nq in (1, 4, 5, 9):
        x = torch.from_numpy(rng.standard_normal((nq, 512))).to(_t(kind))
        x[:, 77] = 1000.0
        got = _run(dev, codes, scales, middles, 64, x, "f32")
        _compare(got, codes, scales, middles, 64, x, "f32")
        # the rows without that weight: no worse than an fp32 sum of what they hold
        small = x.clone()
        small[:, 77] = 0
        _compare(got[:, ::2], codes[::2], scales[::2], middles, 64, small, "f32")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_infinities_and_nan_in_one_vector_stay_in_its_products(dev, kind):
    import torch
    rng = np.random.default_rng(12)
    codes, scales, middles = _case(rng, 40, 130, 32, True)
    codes[:, 5] = np.arange(40) % 15 + 1
    codes[:20, 9] = 8
    x = torch.from_numpy(rng.standard_normal((4, 130))).to(_t(kind))
    x[1, 5], x[2, 9], x[3, 129] = float("inf"), float("-inf"), float("nan")
    got = _run(dev, codes, scales, middles, 32, x, "f32")
    _compare(got[:1], codes, scales, middles, 32, x[:1], "f32")
    with np.errstate(invalid="ignore"):
        want = np.sum(x.double().numpy()[:, None, :] * plain.values(codes, scales, middles, 32)[None], axis=2)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))


def test_products_do_not_change_between_calls_or_with_other_rows_present(dev):
    """The same rows and vectors give the same bits: whatever ran before, and however many rows and vectors stand beside them."""
    import torch
    import vectorstorekit_b200 as vsk
    g = torch.Generator(device="cuda").manual_seed(3)
    q = vsk.Int4Quantizer(dev, 64, False)
    rows = torch.randn((3000, 768), device="cuda", generator=g)
    held = q.quantizeBatch(rows)
    x = torch.randn((6, 768), device="cuda", generator=g)
    first = q.product(x, *held)
    q.product(torch.randn((50, 768), device="cuda", generator=g), *held)
    assert torch.equal(first, q.product(x, *held))


def test_int4_refusals(dev):
    import torch
    import vectorstorekit_b200 as vsk
    lib, h = dev._lib, dev._h
    q = vsk.Int4Quantizer(dev, 32, True)
    x = torch.randn((4, 64), device="cuda")
    codes, scales, _ = q.quantizeBatch(x)
    with pytest.raises(vsk.InvalidInput):
        q.product(x.cpu(), codes, scales)
    with pytest.raises(vsk.InvalidInput):
        q.product(x, codes.cpu(), scales)
    with pytest.raises(vsk.InvalidInput):
        q.product(x, codes, scales, scales)                      # a symmetric quantiser has no middles
    with pytest.raises(vsk.InvalidInput):
        q.product(x, codes, scales.float())
    with pytest.raises(vsk.DimensionMismatch):
        q.product(x[:, :62], codes, scales)
    with pytest.raises(vsk.DimensionMismatch):
        q.product(x, codes, scales[:, :1])
    with pytest.raises(vsk.DimensionMismatch):
        q.product(x[0], codes, scales)
    with pytest.raises(vsk.EmptyInput):
        q.product(x[:0], codes, scales)
    with pytest.raises(vsk.EmptyInput):
        q.quantizeBatch(x[:0])
    with pytest.raises(vsk.UnsupportedOperation):
        q.product(x, codes, scales, out_dtype=torch.float64)
    with pytest.raises(vsk.UnsupportedOperation):
        q.quantizeBatch(x.double())
    # the C entries by themselves
    from vectorstorekit_b200 import _lib
    p = lambda t: C.c_void_p(t.data_ptr())
    y = torch.empty((4, 4), device="cuda")
    lib.vsk_checked_register(p(y), 64)
    r = _lib.Q4Rows(p(codes), p(scales), None, 32, 2, 4, 64, 32)

    def product(**kw):
        a = dict(x=p(x), xt=0, nq=4, xs=64, y=p(y), yt=0, ys=4)
        a.update({k: v for k, v in kw.items() if k in a})
        rr = _lib.Q4Rows(p(codes), p(scales), None, 32, 2, 4, 64, 32)
        for k, v in kw.items():
            if k not in a:
                setattr(rr, k, v)
        return lib.vsk_q4_product_dev(h, C.byref(rr), a["x"], a["xt"], a["nq"], a["xs"], a["y"], a["yt"], a["ys"])

    assert product() == 0
    for status, kw in ((9, dict(n=0)), (9, dict(n=-1)), (9, dict(nq=0)), (8, dict(dim=0)), (3, dict(group=16)), (3, dict(group=0)),
                       (7, dict(codes=None)), (7, dict(scales=None)), (4, dict(code_stride=31)), (4, dict(scale_stride=1)), (3, dict(xt=3)),
                       (3, dict(yt=-1)), (8, dict(xs=63)), (4, dict(ys=3)), (7, dict(x=None)), (7, dict(y=None)),
                       (7, dict(y=C.c_void_p(y.data_ptr() + 2)))):
        assert product(**kw) == status, kw
    assert lib.vsk_q4_product_dev(h, None, p(x), 0, 4, 64, p(y), 0, 4) == 7
    assert lib.vsk_q4_product_dev(None, C.byref(r), p(x), 0, 4, 64, p(y), 0, 4) == 7
    assert lib.vsk_q4_decode_dev(h, C.byref(r), None) == 7
    assert lib.vsk_q4_decode_dev(h, C.byref(r), C.c_void_p(y.data_ptr() + 2)) == 7
    assert lib.vsk_q4_encode_dev(h, p(x), 0, 4, 64, 64, 32, 0, p(codes), 32, p(scales), None) == 7      # middles missing
    assert lib.vsk_q4_encode_dev(h, p(x), 0, 4, 64, 63, 32, 1, p(codes), 32, p(scales), None) == 4
    assert lib.vsk_q4_encode_dev(h, p(x), 0, 4, 64, 64, 32, 1, p(codes), 31, p(scales), None) == 4
    assert product() == 0
