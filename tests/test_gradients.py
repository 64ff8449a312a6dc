"""The global norm of a list of gradients and clipping by it (gloo_amd.Gradients)
against float64 arithmetic.

Tolerances.  The sum runs in float64: n terms, each squared exactly (float32 and
shorter) or with one rounding (float64), so S is within (n + 1) 2^-53 of itself
in any order, and the norm, rounded once to float32, within 2^-24 more.  A clipped
value is x * c: c rounded to float32 and the product rounded to float32 (2^-24
each; for float64 a few 2^-53), then to the tensor's type (half a step, or half
the smallest subnormal)."""
import ctypes
import os
import subprocess
import threading

import numpy as np
import pytest

import gloo_amd
from gloo_amd import Gradients, _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
INF = float("inf")

DTYPES = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16,
          "bf16": torch.bfloat16}
CODES = {torch.float32: 5, torch.float64: 6, torch.float16: 7, torch.bfloat16: 8}


def exact_power(tensors, p):
    flat = [t.detach().cpu().double().numpy().reshape(-1) for t in tensors if t.numel()]
    v = np.abs(np.concatenate(flat)) if flat else np.zeros(0)
    if p == INF:
        return float(v.max()) if v.size else 0.0
    return float(np.sum(v.astype(np.longdouble) ** int(p)))


def exact_norm(tensors, p):
    s = exact_power(tensors, p)
    return float(np.sqrt(np.longdouble(s))) if p == 2 else s


def check_norm(got, tensors, p):
    exp = exact_norm(tensors, p)
    n = sum(t.numel() for t in tensors)
    rel = (n + 3) * 2.0 ** -53 + (2.0 ** -24 if got.dtype == torch.float32 else 0)
    assert abs(float(got) - exp) <= rel * exp, (float(got), exp)


def clip_error(exp, dtype, n):
    """n: terms of the norm, whose own error is part of a float64 result's."""
    f = torch.finfo(dtype)
    if dtype == torch.float64:
        return (n + 8) * 2.0 ** -53 * np.abs(exp) + 2.0 ** -1074
    calc = 2.0 ** -23 * 1.001
    step = 0 if dtype == torch.float32 else f.eps / 2 * 1.001
    return (calc + step) * np.abs(exp) + f.smallest_normal * f.eps / 2


def check_clipped(out, x, total, max_norm, n=0):
    c = min(1.0, max_norm / (total + 1e-6))
    exp = x.detach().cpu().double().numpy() * c
    got = out.detach().cpu().double().numpy()
    tol = clip_error(exp, x.dtype, n) + 1e-9 * np.abs(exp) * (x.dtype != torch.float64)
    assert np.all(np.abs(got - exp) <= tol), np.abs(got - exp).max()


def bucket(sizes, dtype, seed, offset=0, gap=0, scale=0.3):
    """(bucket, views): tensors one after another in one device buffer, from
    `offset` elements on, `gap` elements of 7 between them and around."""
    rng = np.random.default_rng(seed)
    total = offset + sum(sizes) + gap * (len(sizes) + 1) + 64
    b = torch.full((total,), 7.0, dtype=torch.float64)
    at, spans = offset + gap, []
    for s in sizes:
        b[at:at + s] = torch.from_numpy(rng.standard_normal(s) * scale)
        spans.append((at, s))
        at += s + gap
    b = b.to(dtype).cuda()
    return b, [b[i:i + s] for i, s in spans]


def untouched(before, after, views):
    keep = torch.ones(before.numel(), dtype=torch.bool, device="cuda")
    for v in views:
        at = v.storage_offset()
        keep[at:at + v.numel()] = False
    return torch.equal(before[keep], after[keep])


# ---- without a GPU -----------------------------------------------------------

def create(ptrs, counts, codes, outs=None):
    n = len(ptrs)
    arr = (ctypes.c_void_p * n)(*ptrs)
    out = None if outs is None else (ctypes.c_void_p * n)(*outs)
    h = _lib.lib.glx_gradients_create(arr, out, (ctypes.c_size_t * n)(*counts),
                                      (ctypes.c_int * n)(*codes), n)
    return gloo_amd.errors.check_handle(h, "create")


@pytest.mark.parametrize("args, message", [
    (([4096], [4], [2]), "floating"),
    (([4096], [4], [99]), "floating"),
    (([None], [4], [5]), "memory"),
    (([4098], [4], [5]), "aligned"),
    (([4097], [4], [8]), "aligned"),
    (([4096], [4], [5], [8194]), "aligned"),
    (([4096], [1 << 62], [5]), "too long"),
    (([4096, 4096], [4, 4], [5, 5]), "0 and 1 share"),
    (([4096, 8192, 4096 + 12], [4, 4, 4], [5, 5, 5]), "0 and 2 share"),
    (([4096, 8192], [4, 4], [5, 5], [4100, 8192]), "gradient and an output"),
    (([4096, 8192], [4, 4], [5, 5], [8192, 4096]), "gradient and an output"),
    (([4096, 8192], [4, 4], [5, 5], [16384, 16384]), "share"),
])
def test_abi_refuses(args, message):
    with pytest.raises(gloo_amd.EnforceNotMet, match=message):
        create(*args)


def test_abi_refuses_null():
    L = _lib.lib
    assert not L.glx_gradients_create(None, None, None, None, 1)
    assert not L.glx_gradients_create(None, None, None, None, -1)
    assert L.glx_gradients_device(None) == -1 and L.glx_gradients_workspace_bytes(None) == 0
    L.glx_gradients_destroy(None)
    for rc in (L.glx_gradients_power_sum(None, 2.0, 8, 8, None),
               L.glx_gradients_norm(None, 2.0, 8, 5, 8, None),
               L.glx_gradients_clip(None, 1.0, 2.0, None, 8, 5, 8, None)):
        assert rc == _lib.ERR_ENFORCE


def test_python_refuses():
    x = torch.zeros(4)
    with pytest.raises(ValueError, match="cpu"):
        Gradients([x])
    with pytest.raises(ValueError, match="outs"):
        Gradients([x], outs=[])
    with pytest.raises(TypeError):
        Gradients([torch.zeros(4, dtype=torch.int32)])


def test_dense_rule():
    from gloo_amd.gradients import _dense
    x = torch.zeros(4, 6, 5)
    assert _dense(x) and _dense(x.permute(2, 0, 1)) and _dense(x[1:3]) and _dense(x[:, :1][:1])
    assert not _dense(x[:, ::2]) and not _dense(x[:, :3]) and not _dense(x[:, :, :1])
    assert not _dense(torch.zeros(1).expand(4)) and _dense(torch.zeros(()))
    assert not _dense(torch.zeros(9).as_strided((3, 3), (1, 1)))


# ---- the norm ----------------------------------------------------------------

LISTS = [[1], [2], [7, 1, 9], [64], [255, 1, 256, 257], [4099, 0, 3], [1000, 16383, 5, 70001],
         [1 << 20, 3, (1 << 18) + 1]]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
def test_norm(dtype, p):
    for i, sizes in enumerate(LISTS):
        for offset in (0, 1, 5):
            _, views = bucket(sizes, DTYPES[dtype], i, offset)
            g = Gradients(views)
            got = g.norm(p)
            assert got.shape == () and got.dtype == (
                torch.float64 if dtype == "f64" else torch.float32)
            check_norm(got, views, p)
            s = g.power_sum(p)
            assert s.dtype == torch.float64
            n = sum(sizes)
            assert abs(float(s) - exact_power(views, p)) <= \
                (n + 1) * 2.0 ** -53 * exact_power(views, p)


@gpu
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
def test_norm_of_mixed_types_and_many(p):
    views = []
    for i, dtype in enumerate(DTYPES.values()):
        views += bucket([1 + 37 * j % 991 for j in range(300)], dtype, i, offset=i)[1]
    views = views[::3] + views[1::3] + views[2::3]
    check_norm(Gradients(views).norm(p), views, p)
    narrow = [v for v in views if v.dtype != torch.float64]
    assert Gradients(narrow).norm(p).dtype == torch.float32
    check_norm(Gradients(narrow).norm(p), narrow, p)


@gpu
def test_norm_is_the_same_bits_every_time():
    _, views = bucket([100003, 7, 250000], torch.float32, 3, 1)
    g, h = Gradients(views), Gradients(views)
    sums = {float(g.power_sum()) for _ in range(5)} | {float(h.power_sum()) for _ in range(5)}
    assert len(sums) == 1


@gpu
@pytest.mark.parametrize("value, dtype", [
    (1e30, torch.float32), (3e38, torch.bfloat16), (1e-30, torch.float32),
    (1e-45, torch.float32), (6e-8, torch.float16), (65504.0, torch.float16),
    (1e-40, torch.bfloat16), (1e-150, torch.float64)])
def test_norm_neither_overflows_nor_vanishes(value, dtype):
    """Squares beyond float32's range on either side; the norm itself fits, but
    for 70001 times 3e38, whose power sum still does."""
    x = torch.full((70001,), value, dtype=torch.float64).to(dtype).cuda()
    g = Gradients([x])
    assert abs(float(g.power_sum()) / exact_power([x], 2) - 1) <= 70003 * 2.0 ** -53
    n = float(g.norm())
    exp = exact_norm([x], 2)
    if exp > torch.finfo(torch.float32).max:
        assert n == INF
    else:
        # Rounded once to float32: half a step is 2^-24 of a normal value and
        # 2^-150 of a subnormal one (steps of 2^-149), as 70001 times 2^-149 gives
        # (norm 264.58 * 2^-149, of which float32 has 265: 0.42 steps off).
        assert abs(n - exp) <= 2.0 ** -24 * 1.01 * exp + 2.0 ** -150


@gpu
@pytest.mark.parametrize("n", [3, 70001])
def test_range_of_float64_squares(n):
    """p = 2: values whose squares leave float64's range make S infinite or 0, and
    the clip follows; on this side of the range, and for p = 1 and inf, all is well."""
    def grads(value):
        return [torch.full((n,), value, device="cuda", dtype=torch.float64)]
    big, small = grads(1.4e154), grads(1e-163)
    g = Gradients(big)
    assert float(g.power_sum()) == float(g.norm()) == INF
    for p in (1.0, INF):
        check_norm(g.norm(p), big, p)
    assert float(g.clip_norm(1.0)) == INF and not bool(big[0].any())
    g = Gradients(small)
    assert float(g.power_sum()) == float(g.norm()) == 0
    for p in (1.0, INF):
        check_norm(g.norm(p), small, p)
    assert float(g.clip_norm(1.0)) == 0 and bool((small[0] == 1e-163).all())
    for value in (1.3e154 / n ** 0.5, 1e-153):  # squares and their sum are normal values
        x = grads(value)
        check_norm(Gradients(x).norm(), x, 2)
    x = grads(1.3e154 / n ** 0.5)
    was, total = x[0].clone(), exact_norm(x, 2)
    Gradients(x).clip_norm(1.0)
    check_clipped(x[0], was, total, 1.0, n)


@gpu
@pytest.mark.parametrize("n", [3, 70001])
def test_clip_by_a_subnormal_coefficient(n):
    """The coefficient is held in float32: below 2^-126 it is off by up to 2^-150,
    half a step, so that the clipped value x * c is off by |x| 2^-150 beside the
    roundings of every clip."""
    x = torch.full((n,), 1e38, device="cuda")
    x[1::2] = -3e37
    was, total = x.clone(), exact_norm([x], 2)
    for max_norm in (1e-3, 1e-6, 30.0):  # coefficients of 1e-41 and 1e-44 / sqrt(n), and more
        out = torch.empty_like(x)
        Gradients([x], outs=[out]).clip_norm(max_norm)
        w = was.cpu().double().numpy()
        exp = w * (max_norm / (total + 1e-6))
        tol = clip_error(exp, torch.float32, n) + np.abs(w) * 2.0 ** -150
        assert np.all(np.abs(out.cpu().double().numpy() - exp) <= tol)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
def test_norm_not_finite(dtype, p):
    for at in (0, 1, 5000, 99999, 100002):
        _, (x, y) = bucket([100003, 9], DTYPES[dtype], 1, 1)
        x[at] = -INF
        assert float(Gradients([x, y]).norm(p)) == INF
        y[8] = float("nan")
        assert np.isnan(float(Gradients([x, y]).norm(p)))
        assert np.isnan(float(Gradients([x, y]).power_sum(p)))


@gpu
def test_norm_of_nothing():
    assert float(Gradients([]).norm()) == 0
    e = torch.empty(0, device="cuda")
    g = Gradients([e, e])
    assert float(g.norm(INF)) == 0 and float(g.power_sum(1)) == 0
    assert float(g.clip_norm(1.0)) == 0
    assert float(Gradients([torch.zeros(5, device="cuda")]).norm()) == 0
    assert float(Gradients([torch.tensor(-3.0, device="cuda")]).norm()) == 3


@gpu
def test_strides():
    x = torch.randn(6, 70, 11, device="cuda")
    y = torch.randn(2, 3, 8, 8, device="cuda").to(memory_format=torch.channels_last)
    views = [x.permute(2, 0, 1), y, x.new_tensor([2.0]).expand(1, 1)]
    check_norm(Gradients(views).norm(), views, 2)
    outs = [torch.empty_like(v) for v in views]
    total = Gradients(views, outs=outs).clip_norm(0.5)
    for o, v in zip(outs, views):
        check_clipped(o, v, exact_norm(views, 2), 0.5)
    assert abs(float(total) - exact_norm(views, 2)) <= 1e-6 * float(total)
    for bad in (x[:, ::2], x[:, :9], x[:, :, 0], x.new_zeros(1).expand(7)):
        with pytest.raises(ValueError, match="gaps"):
            Gradients([bad])
    with pytest.raises(ValueError, match="strides"):
        Gradients([x], outs=[torch.empty(11, 70, 6, device="cuda").permute(2, 1, 0)])


@gpu
def test_offsets_beyond_32_bits():
    n = (1 << 32) + 77
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    spots = [0, (1 << 31) + 3, (1 << 32) - 1, 1 << 32, n - 1]
    for i, at in enumerate(spots):
        x[at] = 2.0 ** i
    want = sum(4.0 ** i for i in range(len(spots)))
    g = Gradients([x])
    assert float(g.power_sum()) == want
    g.clip_norm(float(np.sqrt(want)) / 2)
    got = [float(x[at]) for at in spots]
    # 1e-6 beside the norm, then bf16's half step
    assert np.allclose(got, [2.0 ** i / 2 for i in range(len(spots))], rtol=2.0 ** -8 + 1e-5, atol=0)
    assert int(x.count_nonzero()) == len(spots)


# ---- clipping ----------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("inplace", [True, False])
def test_clip(dtype, p, inplace):
    for i, sizes in enumerate(LISTS):
        for offset in (0, 1, 5):
            b, views = bucket(sizes, DTYPES[dtype], i, offset, gap=3)
            was = [v.clone() for v in views]
            before = b.clone()
            total = exact_norm(was, p)
            if inplace:
                g, outs, ob, obefore = Gradients(views), views, b, before
            else:
                ob, outs = bucket(sizes, DTYPES[dtype], 99, (offset + 2) % 4, gap=5)
                obefore = ob.clone()
                g = Gradients(views, outs=outs)
            got = g.clip_norm(total / 3, p)
            check_norm(got, was, p)
            assert untouched(obefore, ob, outs)
            if not inplace:
                assert torch.equal(b, before)
            for o, w in zip(outs, was):
                check_clipped(o, w, total, total / 3, sum(sizes))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
def test_clip_below_the_limit_changes_nothing(dtype):
    b, views = bucket([1000, 3, 70001], DTYPES[dtype], 2, 1)
    before = b.clone()
    for limit in (1e6, INF):
        Gradients(views).clip_norm(limit)
        assert torch.equal(b, before)
        ob, outs = bucket([1000, 3, 70001], DTYPES[dtype], 5, 2)
        Gradients(views, outs=outs).clip_norm(limit)
        assert all(torch.equal(o, v) for o, v in zip(outs, views))


@gpu
def test_clip_to_zero():
    _, views = bucket([1000, 3], torch.float32, 2, 1)
    Gradients(views).clip_norm(0.0)
    assert all(int(v.count_nonzero()) == 0 for v in views)
    Gradients(views).clip_norm(0.0)  # 0 / 1e-6
    assert all(int(v.count_nonzero()) == 0 for v in views)


@gpu
def test_clip_not_finite():
    """As 64-bit arithmetic has it: an infinite norm gives 0 (NaN where the
    gradient is infinite), a NaN gives NaN everywhere."""
    x = torch.ones(5000, device="cuda")
    x[77] = INF
    y = torch.ones(9, device="cuda", dtype=torch.bfloat16)
    assert float(Gradients([x, y]).clip_norm(1.0)) == INF
    assert torch.isnan(x[77]) and int(x.nan_to_num(0).count_nonzero()) == 0
    assert int(y.count_nonzero()) == 0
    x.fill_(1)
    x[4999] = float("nan")
    y.fill_(1)
    assert np.isnan(float(Gradients([x, y]).clip_norm(1.0)))
    assert bool(torch.isnan(x).all()) and bool(torch.isnan(y).all())


@gpu
@pytest.mark.parametrize("n", [5000, 1 << 20])  # one launch, and two
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("given", [False, True])
def test_clip_of_an_infinite_norm_by_an_infinite_limit(n, inplace, given):
    """min(1, inf / inf) is NaN; a finite norm is below the limit."""
    x = torch.ones(n, device="cuda")
    x[n // 2] = INF
    y = torch.ones(9, device="cuda", dtype=torch.bfloat16)
    outs = [x, y] if inplace else [torch.zeros_like(x), torch.zeros_like(y)]
    g = Gradients([x, y], outs=outs)
    s = g.power_sum() if given else None
    assert float(g.clip_norm(INF, power_sum=s)) == INF
    assert all(bool(torch.isnan(o).all()) for o in outs)
    x.fill_(2)
    y.fill_(2)
    s = g.power_sum() if given else None
    assert float(g.clip_norm(INF, power_sum=s)) > 2
    assert all(bool((o == 2).all()) for o in outs)


@gpu
def test_clip_by_a_given_power_sum():
    _, views = bucket([1000, 70001], torch.float32, 2, 1)
    was = [v.clone() for v in views]
    s = torch.tensor(400.0, dtype=torch.float64, device="cuda")
    assert float(Gradients(views).clip_norm(5.0, power_sum=s)) == 20
    for v, w in zip(views, was):
        check_clipped(v, w, 20.0, 5.0)
    s.fill_(3.0)
    assert float(Gradients(views).clip_norm(5.0, 1, power_sum=s)) == 3


@gpu
def test_out_arguments():
    x = torch.full((10,), 2.0, device="cuda")
    g = Gradients([x])
    out = torch.zeros(1, device="cuda")
    assert g.norm(INF, out=out) is out and float(out) == 2
    with pytest.raises(ValueError, match="out"):
        g.norm(out=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="out"):
        g.norm(out=torch.zeros(1, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="power_sum"):
        g.clip_norm(1.0, power_sum=out)
    for p in (3.0, 0.0, -INF, float("nan")):
        with pytest.raises(gloo_amd.EnforceNotMet, match="norm is 1, 2"):
            g.norm(p)
    for m in (-1.0, float("nan")):
        with pytest.raises(gloo_amd.EnforceNotMet, match="max_norm"):
            g.clip_norm(m)
    with pytest.raises(gloo_amd.EnforceNotMet, match="share memory"):
        Gradients([x, x])
    with pytest.raises(gloo_amd.EnforceNotMet, match="share memory"):
        Gradients([x[:6], x[5:]])
    with pytest.raises(TypeError):
        Gradients([x], outs=[x.half()])
    with pytest.raises(gloo_amd.EnforceNotMet, match="not a device pointer"):
        host = np.zeros(8, np.float32)
        create([host.ctypes.data], [8], [5])
    g.close()
    with pytest.raises(ValueError, match="closed"):
        g.norm()


@gpu
@pytest.mark.parametrize("n", [10, 1 << 20])  # one workgroup, and many
def test_scalars_apart_from_the_tensors(n):
    """What a call writes beside the tensors lies outside what it reads."""
    x = torch.ones(n, device="cuda", dtype=torch.float64)
    g = Gradients([x[1:-1]])
    s = g.power_sum()
    for out in (x[1], x[n // 2], x[n - 2]):
        with pytest.raises(gloo_amd.EnforceNotMet, match="lies in a tensor"):
            g.norm(out=out)
        with pytest.raises(gloo_amd.EnforceNotMet, match="lies in a tensor"):
            g.clip_norm(1.0, power_sum=out)
    with pytest.raises(gloo_amd.EnforceNotMet, match="share memory"):
        g.clip_norm(1.0, power_sum=s, out=s)
    assert float(g.norm(out=x[0])) == float(g.norm(out=x[n - 1])) == float(np.sqrt(n - 2.0))
    ws = torch.zeros(1 << 14, device="cuda", dtype=torch.float64)
    if _lib.lib.glx_gradients_workspace_bytes(g._h):
        for at in (None, ws.data_ptr() + 4):
            assert _lib.lib.glx_gradients_norm(g._h, 2.0, s.data_ptr(), 6, at, None) == \
                _lib.ERR_ENFORCE
        assert _lib.lib.glx_gradients_norm(g._h, 2.0, ws.data_ptr() + 8, 6, ws.data_ptr(),
                                           None) == _lib.ERR_ENFORCE
    assert _lib.lib.glx_gradients_norm(g._h, 2.0, s.data_ptr(), 5 + 2, ws.data_ptr(), None) == \
        _lib.ERR_ENFORCE
    host = np.zeros(1 << 14)
    for call in (lambda: _lib.lib.glx_gradients_norm(g._h, 2.0, host.ctypes.data, 6,
                                                     ws.data_ptr(), None),
                 lambda: _lib.lib.glx_gradients_clip(g._h, 1.0, 2.0, host.ctypes.data, None, 0,
                                                     None, None)):
        assert call() == _lib.ERR_ENFORCE and "not a device pointer" in _lib.last_error()
    assert bool((x[1:-1] == 1).all())
    # no norm wanted: the clip alone
    assert _lib.lib.glx_gradients_clip(g._h, 0.5, float("inf"), None, None, 0, ws.data_ptr(),
                                       None) == 0
    torch.cuda.synchronize()
    assert bool(((x[1:-1] - 0.5).abs() <= 1e-6).all()) and float(x[0]) != 0.5


@gpu
def test_workspace_apart_from_the_tensors():
    """By the C ABI, on the host: a workspace in a gradient, or in host memory."""
    x = torch.ones(1 << 20, device="cuda")
    out = torch.zeros(1, device="cuda")
    g = Gradients([x])
    assert _lib.lib.glx_gradients_workspace_bytes(g._h) > 0
    host = np.zeros(1 << 14)
    for ws, message in ((x.data_ptr() + 4096, "workspace lies in a tensor"),
                        (host.ctypes.data, "not a device pointer")):
        for call in (lambda: _lib.lib.glx_gradients_norm(g._h, 2.0, out.data_ptr(), 5, ws, None),
                     lambda: _lib.lib.glx_gradients_clip(g._h, 1.0, 2.0, None, None, 0, ws, None)):
            with pytest.raises(gloo_amd.EnforceNotMet, match=message):
                gloo_amd.errors.check(call())
    torch.cuda.synchronize()
    assert bool((x == 1).all()) and float(out) == 0 and not host.any()


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_clip_of_subnormal_values(dtype):
    """Values down to the type's smallest, clipped by a norm that one large value
    makes: rounded to the subnormal grid, not flushed."""
    t = DTYPES[dtype]
    f = torch.finfo(t)
    tiny = f.smallest_normal * f.eps
    v = torch.arange(1, 3000, dtype=torch.float64) * tiny
    x = torch.cat([v, -v, torch.tensor([4.0], dtype=torch.float64)]).to(t).cuda()
    was = x.clone()
    total = exact_norm([was], 2)
    out = torch.empty_like(x)
    Gradients([x], outs=[out]).clip_norm(total / 3)
    check_clipped(out, was, total, total / 3)
    assert int(out.count_nonzero()) > 5000 - 4


@gpu
def test_negated_views_are_refused():
    x = torch._neg_view(torch.ones(8, device="cuda"))
    for call in (lambda: Gradients([x]), lambda: gloo_amd.mx.quantize(x)):
        with pytest.raises(ValueError, match="negated"):
            call()


@gpu
def test_keeps_the_memory_it_was_given():
    """A parameter whose gradient is replaced: the handle still has the old one."""
    w = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
    w.grad = torch.full((1000,), 2.0, device="cuda")
    g = Gradients([w.grad])
    w.grad = None
    fresh = [torch.full((1000,), 5.0, device="cuda") for _ in range(8)]
    assert abs(float(g.norm()) - np.sqrt(4000)) < 1e-4
    assert all(float(f[0]) == 5 for f in fresh)


# ---- streams and graphs ------------------------------------------------------

@gpu
def test_streams():
    _, views = bucket([100003, 5], torch.bfloat16, 3, 1)
    g = Gradients(views)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for stream in (s, s.cuda_stream, torch.cuda.default_stream()):
        n = g.norm(stream=stream)
        torch.cuda.synchronize()
        check_norm(n, views, 2)
    with torch.cuda.stream(s):  # the default stream by its handle, from another current one
        n = g.norm(stream=0)
    torch.cuda.synchronize()
    check_norm(n, views, 2)


@gpu
def test_object_dropped_while_its_work_is_queued():
    """Dropping the object waits for the device before its table goes."""
    x = torch.ones(1 << 20, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        n = Gradients([x]).norm()
        fresh = [torch.full((64,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    assert float(n) == 1024 and len(fresh) == 64


@gpu
def test_close_waits_for_queued_work():
    """What the handle promises: after close() nothing reads its table any more."""
    g = Gradients([torch.ones(1 << 20, device="cuda")])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)
        n = g.norm()
    assert not s.query()
    g.close()
    assert s.query()
    assert float(n) == 1024


@gpu
@pytest.mark.parametrize("mode", ["global", "thread_local"])
@pytest.mark.parametrize("thread", [False, True])
def test_dropped_while_a_graph_is_captured(mode, thread):
    """An object that the graph does not hold, dropped by the garbage collector
    or another thread in the middle of a capture: the capture goes on."""
    x = torch.zeros(1 << 16, device="cuda")
    old = Gradients([torch.ones(1 << 16, device="cuda")])
    g = Gradients([x])
    old.norm(), g.norm()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(), capture_error_mode=mode):
        x.add_(1)
        if thread:
            t = threading.Thread(target=old.close)
            t.start()
            t.join()
        else:
            old.close()
        n = g.norm()
    for step in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert float(n) == 256 * step and float(g.norm()) == 256 * step


@gpu
def test_two_streams_at_once():
    """One handle, two streams, many calls in flight: every result is right."""
    _, views = bucket([3000017, 5], torch.float32, 3, 1)
    g = Gradients(views)
    want = float(g.power_sum())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [g.power_sum(stream=streams[i % 2]) for i in range(40)]
    torch.cuda.synchronize()
    assert {float(v) for v in got} == {want}


@gpu
def test_graph_replays():
    """Two captured graphs of one handle, replayed in turn and at once with
    eager calls between: every replay equals the eager result."""
    b, views = bucket([200003, 5, 40000], torch.float32, 3, 1)
    outs = [torch.empty_like(v) for v in views]
    g = Gradients(views, outs=outs)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, results = [], []
    for s, fn in zip(streams, (lambda: g.clip_norm(0.5), lambda: g.norm(1.0))):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            results.append(fn())
        graphs.append(graph)
    for step in range(4):
        for i, v in enumerate(views):
            v.normal_(generator=torch.Generator("cuda").manual_seed(10 * step + i))
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        check_norm(results[0], views, 2)
        check_norm(results[1], views, 1)
        for o, v in zip(outs, views):
            check_clipped(o, v, exact_norm(views, 2), 0.5)
        eager = [torch.empty_like(v) for v in views]
        assert float(Gradients(views, outs=eager).clip_norm(0.5)) == float(results[0])
        assert all(torch.equal(a, c) for a, c in zip(eager, outs))


# ---- with the rest of the framework ------------------------------------------

def test_header_wrappers_compile(tmp_path):
    """gloo_amd.hpp's Gradients and mx over the same entry points."""
    build_cpp(str(tmp_path / "gradients_test"))


def build_cpp(out):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "gloo_amd")
    subprocess.check_call(
        ["g++", "-std=c++17", "-O2", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
         "-I" + os.path.join(root, "include"),
         os.path.join(root, "tests", "cpp", "gradients_test.cc"), "-o", out, "-L" + lib,
         "-lgloo_amd", "-L/opt/rocm/lib", "-lamdhip64", "-lpthread", "-Wl,-rpath," + lib])


@gpu
def test_header_wrappers_run(tmp_path):
    exe = str(tmp_path / "gradients_test")
    build_cpp(exe)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "all passed" in p.stdout, p.stdout + p.stderr


@gpu
@pytest.mark.parametrize("p", [2.0, INF])
def test_sharded_gradients_of_ranks(p):
    """Three thread-ranks hold shards: the power sums go through the framework's
    allreduce (SUM, MAX for inf) and every rank clips by the global norm."""
    P = 3
    shards = [bucket([4099 + r, 7, 30001], (torch.float32, torch.bfloat16)[r % 2], r, r)[1]
              for r in range(P)]
    was = [[v.clone() for v in s] for s in shards]
    torch.cuda.synchronize()
    store = gloo_amd.rendezvous.HashStore()
    norms, errs = [None] * P, []

    def rank(r):
        try:
            torch.cuda.set_device(0)
            ctx = gloo_amd.rendezvous.Context(r, P, 0)
            ctx.setTimeout(60)
            ctx.connectFullMesh(store)
            g = Gradients(shards[r])
            s = g.power_sum(p).reshape(1)
            torch.cuda.current_stream().synchronize()
            fn = gloo_amd.ReductionFunction.max if p == INF else gloo_amd.ReductionFunction.sum
            ar = gloo_amd.AllreduceRingChunked(ctx, [s], fn=fn)
            ar.run()
            norms[r] = float(g.clip_norm(1.0, p, power_sum=s))
            torch.cuda.synchronize()
            ar.close()
        except BaseException as e:  # noqa: BLE001
            errs.append(e)

    ts = [threading.Thread(target=rank, args=(r,)) for r in range(P)]
    [t.start() for t in ts]
    [t.join(120) for t in ts]
    assert not errs, errs
    every = [v for s in was for v in s]
    total = exact_norm(every, p)
    for r in range(P):
        assert abs(norms[r] - total) <= 2.0 ** -23 * total
        for v, w in zip(shards[r], was[r]):
            check_clipped(v, w, total, 1.0)
