"""Microscaled 4-bit messages (gloo_amd.mx) against a plain restatement of the
OCP MX rules in 64 bits (numpy).  Payloads are compared byte for byte: the
operator's arithmetic before its one rounding is exact (powers of two, a sum
held in fp32 as defined), so there is nothing to be off by.  Float results of a
fold are the fp32 left fold's own bits, rounded once to the output's type."""
import ctypes
import threading

import numpy as np
import pytest

import gloo_amd
from gloo_amd import _lib, mx

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

FP4 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
MID = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5])  # where two codes meet
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def blocks_of(v):
    n = v.size
    nb = -(-n // 32)
    b = np.zeros(nb * 32, v.dtype)
    b[:n] = v
    return b.reshape(nb, 32)


def payload_of(y):
    """(payload bytes, values in float64) of float32 values y."""
    y = np.asarray(y, np.float32)
    b = blocks_of(y)
    nb = b.shape[0]
    with np.errstate(invalid="ignore"):
        wide = np.abs(b.astype(np.float64))
        top = wide.max(axis=1) if nb else np.zeros(0)
    bad = ~np.isfinite(top)
    _, e = np.frexp(np.where(bad | (top == 0), 1.0, top))
    byte = np.where(top == 0, 0, np.maximum(e - 1 + 127 - 2, 0))
    a = np.where(bad[:, None], 0.0, wide) * np.ldexp(1.0, 127 - byte)[:, None]
    code = np.searchsorted(MID, a, side="left")
    for tie in (.75, 1.75, 3.5):  # halfway goes to the code with an even mantissa
        code = np.where(a == tie, np.searchsorted(MID, tie, side="right"), code)
    code = np.where(np.signbit(b), code + 8, code)
    code[bad] = 0
    byte = np.where(bad, 255, byte)
    out = np.zeros(mx_bytes(y.size), np.uint8)
    out[:nb * 16] = (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8).reshape(-1)
    out[nb * 16:nb * 17] = byte
    return out, values_of(out, y.size)


def mx_bytes(n):
    return -(-(-(-n // 32) * 17) // 16) * 16


def values_of(payload, n):
    nb = -(-n // 32)
    c = np.empty(nb * 32, np.int64)
    c[0::2], c[1::2] = payload[:nb * 16] & 15, payload[:nb * 16] >> 4
    s = payload[nb * 16:nb * 17].astype(np.int64)
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (FP4[c].reshape(nb, 32) * scale[:, None]).reshape(-1)[:n]


def fold_of(payloads, n, scale):
    """The left fold in fp32 (each partial sum rounded once), times scale in fp32."""
    with np.errstate(over="ignore", invalid="ignore"):
        acc = values_of(payloads[0], n).astype(np.float32)
        for p in payloads[1:]:
            acc = (acc.astype(np.float64) + values_of(p, n)).astype(np.float32)
        return acc * np.float32(scale)


def same_bits(got, exp):
    got, exp = np.asarray(got), np.asarray(exp)
    nan = np.isnan(exp)
    assert np.array_equal(np.isnan(got), nan)
    view = {4: np.uint32, 2: np.uint16}[exp.dtype.itemsize]
    bad = np.flatnonzero((got.view(view) != exp.view(view)) & ~nan)
    assert bad.size == 0, (bad[:5], got[bad[:5]], exp[bad[:5]])


def as_numpy(t):
    return t.detach().cpu().float().numpy() if t.dtype == torch.bfloat16 else \
        t.detach().cpu().numpy()


def rounded(v, dtype):
    """fp32 values rounded to dtype, as float32 (bf16) or the type itself."""
    with np.errstate(over="ignore"):
        return as_numpy(torch.from_numpy(np.ascontiguousarray(v)).to(dtype))


def gradient(n, seed, dtype=torch.float32):
    """Values of varying magnitude, some blocks of zeros, as a CPU tensor."""
    rng = np.random.default_rng(seed)
    v = rng.standard_normal(n) * np.exp2(rng.integers(-12, 6, n // 50 + 1)).repeat(50)[:n]
    v[n // 3: n // 3 + 40] = 0
    return torch.from_numpy(v.astype(np.float32)).to(dtype)


def random_payload(n, rng, low=100, high=140):
    p = np.zeros(mx_bytes(n), np.uint8)
    nb = -(-n // 32)
    p[:nb * 16] = rng.integers(0, 256, nb * 16)
    p[nb * 16:nb * 17] = rng.integers(low, high, nb)
    return p


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- without a GPU -----------------------------------------------------------

@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 255, 256, 257, 512, 4099, (1 << 33) + 1])
def test_payload_bytes(n):
    assert mx.payload_bytes(n) == mx_bytes(n) == _lib.lib.glx_mx_payload_bytes(n)


def test_payload_bytes_refuses():
    for n in (-1, (1 << 60) + 1):
        with pytest.raises(ValueError):
            mx.payload_bytes(n)


def test_oracle_rounding():
    """The restatement itself: every code, every halfway point."""
    y = np.zeros(32, np.float32)
    y[:17] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -5, 5.5, 1e-9, -0., 7, 7.99, -7]
    p, v = payload_of(y)
    assert p[16] == 127 and list(v[:17]) == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -4, 6, 0, 0, 6, 6, -6]
    assert np.signbit(v[13]) and np.signbit(v[8])


P16 = ctypes.c_void_p * 17


@pytest.mark.parametrize("call, message", [
    (lambda L: L.glx_mx_quantize(6, 4096, 8192, None, None, 4, None), "float32"),
    (lambda L: L.glx_mx_quantize(5, 4096 + 8, 8192, None, None, 4, None), "16-byte"),
    (lambda L: L.glx_mx_quantize(5, None, 8192, None, None, 4, None), "payload"),
    (lambda L: L.glx_mx_quantize(5, 4096, None, None, None, 4, None), "x"),
    (lambda L: L.glx_mx_quantize(5, 4096, 8194, None, None, 4, None), "misaligned"),
    (lambda L: L.glx_mx_quantize(5, 4096, 8192, 16386, None, 4, None), "residual"),
    (lambda L: L.glx_mx_quantize(5, 8208, 8192, None, None, 64, None), "shares"),
    (lambda L: L.glx_mx_quantize(5, 4096, 8192, 16384, 16388, 64, None), "overlap"),
    (lambda L: L.glx_mx_quantize(7, 4096, 8192, None, 8192, 64, None), "overlaps x"),
    (lambda L: L.glx_mx_reduce_n(3, 4096, P16(8192), 1, 4, 1.0, None), "float32"),
    (lambda L: L.glx_mx_reduce_n(5, 4096, P16(8192), 0, 4, 1.0, None), "1..16"),
    (lambda L: L.glx_mx_reduce_n(5, 4096, P16(*[8192] * 17), 17, 4, 1.0, None), "1..16"),
    (lambda L: L.glx_mx_reduce_n(5, 4096, None, 1, 4, 1.0, None), "1..16"),
    (lambda L: L.glx_mx_reduce_n(5, 4096, P16(8192, None), 2, 4, 1.0, None), "payload 1"),
    (lambda L: L.glx_mx_reduce_n(5, 4098, P16(8192), 1, 4, 1.0, None), "misaligned dst"),
    (lambda L: L.glx_mx_reduce_n(5, 4096, P16(4112), 1, 64, 1.0, None), "share"),
    (lambda L: L.glx_mx_reduce_n(5, 4096, P16(8192), 1, 4, float("nan"), None), "finite"),
    (lambda L: L.glx_mx_requantize_n(4096, P16(4112), 1, 64, 1.0, None), "overlaps"),
    (lambda L: L.glx_mx_requantize_n(4104, P16(8192), 1, 64, 1.0, None), "16-byte"),
    (lambda L: L.glx_mx_requantize_n(4096, P16(8192), 1, 64, float("inf"), None), "finite"),
])
def test_abi_refuses(call, message):
    with pytest.raises(gloo_amd.EnforceNotMet, match=message):
        gloo_amd.errors.check(call(_lib.lib))


def test_nothing_to_do_without_gpu():
    assert _lib.lib.glx_mx_quantize(5, None, None, None, None, 0, None) == 0
    assert _lib.lib.glx_mx_reduce_n(5, None, P16(), 1, 0, 1.0, None) == 0
    assert _lib.lib.glx_mx_requantize_n(None, P16(), 1, 0, 1.0, None) == 0


def test_python_refuses_host_tensors():
    x, p = torch.zeros(64), torch.zeros(48, dtype=torch.uint8)
    for call in (lambda: mx.quantize(x, p), lambda: mx.reduce_n(x, [p]),
                 lambda: mx.dequantize(x, p), lambda: mx.requantize_n(p, [p], 64)):
        with pytest.raises(ValueError, match="cpu"):
            call()


# ---- quantisation ------------------------------------------------------------

def check_quantize(x, offset=0, residual=None, want_residual=False, inplace=False):
    """x: CPU tensor.  Runs it from `offset` elements into a buffer, with
    guard bytes around everything written."""
    n = x.numel()
    buf = torch.zeros(offset + n + 64, dtype=x.dtype)
    buf[offset:offset + n] = x
    d = buf.cuda()[offset:offset + n]
    y = x.float().numpy()
    r = None
    if residual is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            y = y + residual
        rbuf = np.full(offset + n + 64, 7, np.float32)
        rbuf[offset:offset + n] = residual
        rdev = dev(rbuf)
        r = rdev[offset:offset + n]
    ro = None
    if want_residual:
        odev = rdev if inplace else torch.full((offset + n + 64,), 7.0, device="cuda")
        ro = odev[offset:offset + n]
    size = mx_bytes(n)
    pay = torch.full((size + 64,), 0xa5, dtype=torch.uint8, device="cuda")
    assert mx.quantize(d, pay, residual=r, residual_out=ro) is pay
    got = pay.cpu().numpy()
    exp, values = payload_of(y)
    bad = np.flatnonzero(got[:size] != exp)
    assert bad.size == 0, (n, bad[:5], got[bad[:5]], exp[bad[:5]])
    assert np.all(got[size:] == 0xa5), "wrote behind the payload"
    if want_residual:
        full = odev.cpu().numpy()
        assert np.all(full[:offset] == 7) and np.all(full[offset + n:] == 7)
        with np.errstate(invalid="ignore"):
            left = np.where(np.isnan(values), 0.0, y.astype(np.float64) - values)
        assert np.array_equal(full[offset:offset + n].astype(np.float64), left)
    out = torch.empty(n, device="cuda")
    mx.dequantize(out, pay)
    same_bits(out.cpu().numpy(), values.astype(np.float32))


SIZES = [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257, 511, 1000, 2047, 4099, 65537]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_quantize_sizes(dtype, offset):
    for n in SIZES:
        check_quantize(gradient(n, n, DTYPES[dtype]), offset)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_quantize_every_value(dtype):
    """All 65536 values of a 16-bit type: in order (neighbours share a block),
    shuffled finite ones (every scale with every smaller value), and each NaN
    and infinity among them."""
    bits = np.arange(65536, dtype=np.uint16)
    x = torch.from_numpy(bits.view(np.int16).copy()).view(dtype)
    check_quantize(x)
    finite = x[torch.isfinite(x)]
    g = torch.Generator().manual_seed(3)
    check_quantize(finite[torch.randperm(finite.numel(), generator=g)], 1, want_residual=True)


@gpu
def test_quantize_halfway_points_at_every_scale():
    """f32: for every exponent of a block's maximum, each code, each halfway
    point and its neighbours, with both signs; subnormal blocks included."""
    rows = []
    for e in range(-126, 128):
        b = np.concatenate([FP4[:8], MID, [7.0, 7.75]]).astype(np.float64)
        v = np.ldexp(b, e - 2).astype(np.float32)
        near = np.concatenate([v, np.nextafter(v, np.float32(0)),
                               np.nextafter(v, np.float32(3e38))])
        near = near[(near < np.ldexp(2.0, e)) & np.isfinite(near)]
        top = np.float32(np.ldexp(1.0, e))
        for sign in (1, -1):
            for part in np.array_split(sign * near, 3):
                row = np.zeros(32, np.float32)
                row[:part.size] = part
                row[31] = top
                rows.append(row)
    tiny = (np.arange(1, 33, dtype=np.uint32)[None, :] << np.arange(0, 20)[:, None]).view(np.float32)
    check_quantize(torch.from_numpy(np.concatenate(rows + [tiny.reshape(-1)])), want_residual=True)


@gpu
def test_quantize_not_finite():
    for bad in (np.inf, -np.inf, np.nan):
        for at in (0, 31, 32, 70, 99):
            x = gradient(100, 5)
            x[at] = bad
            check_quantize(x, 1, residual=np.ones(100, np.float32), want_residual=True)
    big = torch.full((40,), 3e38)  # x + residual overflows in the first block only
    r = np.zeros(40, np.float32)
    r[3] = 3e38
    check_quantize(big, residual=r, want_residual=True)


@gpu
def test_quantize_zero_blocks():
    x = torch.zeros(96)
    x[40] = -0.0
    x[64:] = 1e-44
    check_quantize(x, want_residual=True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("inplace", [False, True])
def test_quantize_feedback(dtype, inplace):
    for n in SIZES:
        r = gradient(n, n + 1).numpy() * np.float32(0.1)
        check_quantize(gradient(n, n, DTYPES[dtype]), n % 4, r, True, inplace)
        check_quantize(gradient(n, n, DTYPES[dtype]), n % 4, r)


@gpu
def test_feedback_into_x():
    """A float32 x may take the residual."""
    x = gradient(3001, 8)
    d = x.cuda()
    pay = mx.quantize(d, residual_out=d)
    exp, values = payload_of(x.numpy())
    assert np.array_equal(pay.cpu().numpy(), exp)
    assert np.array_equal(d.cpu().numpy().astype(np.float64), x.numpy() - values)


@gpu
def test_feedback_keeps_the_sum():
    """Ten messages and the last residual add up to what was fed in: each step
    rounds x + r once (2^-24 of |x + r|), everything else is exact."""
    n = 4099
    err = torch.zeros(n, device="cuda")
    fed, sent, slack = np.zeros(n), np.zeros(n), np.zeros(n)
    for step in range(10):
        x = gradient(n, 100 + step)
        slack += 2.0 ** -24 * (np.abs(x.numpy()) + np.abs(err.cpu().numpy()))
        pay = mx.quantize(x.cuda(), residual=err, residual_out=err)
        fed += x.numpy()
        sent += values_of(pay.cpu().numpy(), n)
    assert np.all(np.abs(sent + err.cpu().numpy() - fed) <= slack)


@gpu
def test_quantize_refuses():
    x = torch.zeros(64, device="cuda")
    p = torch.zeros(48, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="48"):
        mx.quantize(torch.zeros(65, device="cuda"), p)
    with pytest.raises(ValueError, match="contiguous"):
        mx.quantize(torch.zeros(8, 8, device="cuda").t(), p)
    with pytest.raises(TypeError):
        mx.quantize(x, p.view(torch.int8))
    with pytest.raises(TypeError):
        mx.quantize(x, p, residual=x.half())
    with pytest.raises(ValueError, match="elements"):
        mx.quantize(x, p, residual=x[:63])
    with pytest.raises(TypeError, match="float64"):
        mx.quantize(x.double(), p)
    with pytest.raises(gloo_amd.EnforceNotMet, match="16-byte"):
        mx.quantize(x, torch.zeros(64, dtype=torch.uint8, device="cuda")[8:56])
    with pytest.raises(gloo_amd.EnforceNotMet, match="shares"):
        mx.quantize(x, x.view(torch.uint8)[:48])
    host = np.zeros(4096, np.uint8)
    at = host.ctypes.data + -host.ctypes.data % 16
    L, xp, pp = _lib.lib, x.data_ptr(), p.data_ptr()
    for call in (lambda: L.glx_mx_quantize(5, at, xp, None, None, 4, None),
                 lambda: L.glx_mx_reduce_n(5, at, P16(pp), 1, 4, 1.0, None),
                 lambda: L.glx_mx_requantize_n(at, P16(pp), 1, 4, 1.0, None)):
        with pytest.raises(gloo_amd.EnforceNotMet, match="not a device pointer"):
            gloo_amd.errors.check(call())


@gpu
def test_host_memory_is_refused_at_every_pointer():
    """By the C ABI, on the host: nothing is launched.  Pinned memory is not host
    memory in this sense, kernels reach it."""
    x = gradient(64, 3).cuda()
    p = torch.full((48,), 0xa5, dtype=torch.uint8, device="cuda")
    r = torch.zeros(64, device="cuda")
    host = np.zeros(4096, np.uint8)
    at = host.ctypes.data + -host.ctypes.data % 16
    L, xp, pp, rp = _lib.lib, x.data_ptr(), p.data_ptr(), r.data_ptr()
    for call, what in (
            (lambda: L.glx_mx_quantize(5, at, xp, rp, rp, 64, None), "device pointer"),
            (lambda: L.glx_mx_quantize(5, pp, at, rp, rp, 64, None), "x is host"),
            (lambda: L.glx_mx_quantize(5, pp, xp, at, rp, 64, None), "residual is host"),
            (lambda: L.glx_mx_quantize(5, pp, xp, rp, at, 64, None), "residual_out is host"),
            (lambda: L.glx_mx_reduce_n(5, at, P16(pp), 1, 64, 1.0, None), "device pointer"),
            (lambda: L.glx_mx_reduce_n(5, xp, P16(pp, at), 2, 64, 1.0, None), "payload 1 is host"),
            (lambda: L.glx_mx_requantize_n(at, P16(pp), 1, 64, 1.0, None), "device pointer"),
            (lambda: L.glx_mx_requantize_n(pp, P16(at), 1, 64, 1.0, None), "payload 0 is host")):
        with pytest.raises(gloo_amd.EnforceNotMet, match=what):
            gloo_amd.errors.check(call())
    torch.cuda.synchronize()
    assert bool((p == 0xa5).all()) and not bool(r.any()) and not host.any()
    exp, values = payload_of(x.cpu().numpy())
    px = torch.empty(64, pin_memory=True).copy_(x)
    pr = torch.full((64,), 7.0, pin_memory=True)
    torch.cuda.synchronize()
    gloo_amd.errors.check(L.glx_mx_quantize(5, pp, px.data_ptr(), None, pr.data_ptr(), 64, None))
    torch.cuda.synchronize()
    assert np.array_equal(p.cpu().numpy(), exp)
    assert np.array_equal(pr.numpy().astype(np.float64), x.cpu().numpy() - values)


# ---- the fold ----------------------------------------------------------------

@gpu
@pytest.mark.parametrize("k", list(range(1, 17)))
def test_reduce_n(k):
    rng = np.random.default_rng(k)
    for n in (1, 33, 1000, 4099 + k):
        pays = [random_payload(n, rng) for _ in range(k)]
        for scale in (1.0, 1.0 / k, -0.75):
            exp = fold_of(pays, n, scale)
            for dtype in DTYPES.values():
                buf = torch.full((n + 70,), 7.0, dtype=dtype, device="cuda")
                off = (n + k) % 3
                mx.reduce_n(buf[off:off + n], [dev(p) for p in pays], scale=scale)
                got = as_numpy(buf)
                assert np.all(got[:off] == 7) and np.all(got[off + n:] == 7)
                same_bits(got[off:off + n], rounded(exp, dtype))


@gpu
@pytest.mark.parametrize("k", [1, 2, 3, 8, 16])
def test_requantize_n(k):
    rng = np.random.default_rng(50 + k)
    for n in SIZES:
        pays = [random_payload(n, rng) for _ in range(k)]
        exp, _ = payload_of(fold_of(pays, n, 0.5))
        ds = [dev(p) for p in pays]
        out = torch.full((mx_bytes(n) + 64,), 0xa5, dtype=torch.uint8, device="cuda")
        mx.requantize_n(out, ds, n, scale=0.5)
        got = out.cpu().numpy()
        assert np.array_equal(got[:exp.size], exp) and np.all(got[exp.size:] == 0xa5)
        mx.requantize_n(ds[-1], ds, n, scale=0.5)  # over one of its sources
        assert np.array_equal(ds[-1].cpu().numpy(), exp)


@gpu
def test_fold_every_scale_byte():
    """Scale bytes 0 (subnormal results), up to 252 (the largest a message has),
    253 and 254 (hand-made: beyond float32), 255 (NaN)."""
    n = 256 * 32
    rng = np.random.default_rng(9)
    p = random_payload(n, rng)
    p[n // 2:n // 2 + 256] = np.arange(256)
    q = random_payload(n, rng)
    out = torch.empty(n, device="cuda")
    mx.dequantize(out, dev(p))
    with np.errstate(over="ignore"):
        same_bits(out.cpu().numpy(), values_of(p, n).astype(np.float32))
    mx.reduce_n(out, [dev(q), dev(p)])
    same_bits(out.cpu().numpy(), fold_of([q, p], n, 1.0))
    again = torch.empty(mx_bytes(n), dtype=torch.uint8, device="cuda")
    mx.requantize_n(again, [dev(p)], n)
    with np.errstate(over="ignore"):
        exp, _ = payload_of(values_of(p, n).astype(np.float32))
    assert np.array_equal(again.cpu().numpy(), exp)


@gpu
def test_fold_order_is_left_to_right():
    """Scales far apart: only the left fold gives these bits."""
    rng = np.random.default_rng(4)
    n = 4096
    pays = [random_payload(n, rng, 127 + 12 * ((j * 5) % 7), 128 + 12 * ((j * 5) % 7))
            for j in range(7)]
    out = torch.empty(n, device="cuda")
    mx.reduce_n(out, [dev(p) for p in pays])
    same_bits(out.cpu().numpy(), fold_of(pays, n, 1.0))
    assert not np.array_equal(fold_of(pays, n, 1.0), fold_of(pays[::-1], n, 1.0))


@gpu
def test_fold_reads_nothing_behind_the_end():
    """Codes behind element n - 1 of a source, and bytes behind its scales, do
    not reach the result."""
    rng = np.random.default_rng(6)
    for n in (1, 5, 33, 4099):
        p = random_payload(n, rng)
        clean = p.copy()
        nb = -(-n // 32)
        codes = np.stack([clean[:nb * 16] & 15, clean[:nb * 16] >> 4], 1).reshape(-1)
        codes[n:] = 0
        clean[:nb * 16] = codes[0::2] | (codes[1::2] << 4)
        long = np.concatenate([p, np.full(32, 0xff, np.uint8)])
        long[nb * 17:] = 0xff
        out = torch.empty(mx_bytes(n), dtype=torch.uint8, device="cuda")
        mx.requantize_n(out, [dev(long)], n)
        exp, _ = payload_of(values_of(clean, n).astype(np.float32))
        assert np.array_equal(out.cpu().numpy(), exp)


@gpu
def test_fold_refuses():
    x = torch.zeros(64, device="cuda")
    p = torch.zeros(48, dtype=torch.uint8, device="cuda")
    with pytest.raises(gloo_amd.EnforceNotMet, match="1..16"):
        mx.reduce_n(x, [])
    with pytest.raises(gloo_amd.EnforceNotMet, match="1..16"):
        mx.reduce_n(x, [p] * 17)
    with pytest.raises(ValueError, match="payload 1"):
        mx.reduce_n(x, [p, p[:32]])
    with pytest.raises(gloo_amd.EnforceNotMet, match="share"):
        mx.reduce_n(x, [x.view(torch.uint8)[:48]])
    with pytest.raises(gloo_amd.EnforceNotMet, match="finite"):
        mx.reduce_n(x, [p], scale=float("nan"))
    with pytest.raises(TypeError, match="float64"):
        mx.reduce_n(x.double(), [p])
    with pytest.raises(ValueError, match="bytes"):
        mx.requantize_n(p, [p], 128)


# ---- streams, graphs, length -------------------------------------------------

@gpu
def test_streams():
    """On a stream that is not the current one, as an object and as a raw handle."""
    x = gradient(100003, 1)
    d = x.cuda()
    exp, values = payload_of(x.numpy())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for stream in (s, s.cuda_stream):
        pay = mx.quantize(d, stream=stream)
        out = torch.empty(100003, device="cuda")
        mx.dequantize(out, pay, stream=stream)
        s.synchronize()
        assert np.array_equal(pay.cpu().numpy(), exp)
        same_bits(out.cpu().numpy(), values.astype(np.float32))


@gpu
def test_graph_replays():
    """Quantise with feedback, fold and requantise, captured; every replay on new
    values equals the eager calls."""
    n = 50021
    x = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(n, device="cuda")
    pay, other, hop = (torch.zeros(mx_bytes(n), dtype=torch.uint8, device="cuda")
                       for _ in range(3))
    out = torch.empty(n, device="cuda")
    x.copy_(gradient(n, 0).cuda())
    other.copy_(mx.quantize(gradient(n, 99).cuda()))
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        mx.quantize(x, pay, residual=err, residual_out=err)
        mx.requantize_n(hop, [pay, other], n, scale=0.5)
        mx.reduce_n(out, [hop, pay])
    want = np.zeros(n, np.float32)
    for step in range(4):
        v = gradient(n, step, torch.bfloat16)
        x.copy_(v)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        y = v.float().numpy() + want
        p, values = payload_of(y)
        want = (y - values).astype(np.float32)
        h, _ = payload_of(fold_of([p, other.cpu().numpy()], n, 0.5))
        assert np.array_equal(pay.cpu().numpy(), p)
        assert np.array_equal(hop.cpu().numpy(), h)
        same_bits(out.cpu().numpy(), fold_of([h, p], n, 1.0))
        eager = mx.quantize(v.cuda())
        assert np.array_equal(eager.cpu().numpy(), payload_of(v.float().numpy())[0])


def check_windows(x, y, spots, pay, out, n):
    """Payload and values of x + residual = y in windows [at, at + m) that start
    at blocks: y is a function of (at, m)."""
    nb = -(-n // 32)
    for at, m in spots:
        exp, values = payload_of(y(at, m))
        k = -(-m // 32)
        assert np.array_equal(pay[at // 2:at // 2 + k * 16].cpu().numpy(), exp[:k * 16])
        sc = nb * 16 + at // 32
        assert np.array_equal(pay[sc:sc + k].cpu().numpy(), exp[k * 16:k * 17])
        same_bits(as_numpy(out[at:at + m]), rounded(values.astype(np.float32), out.dtype))


@gpu
def test_offsets_beyond_32_bits():
    """2^32 + 77 elements: windows at the start, around 2^31 and 2^32, and the end."""
    n = (1 << 32) + 77
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    spots = [(0, 4096), ((1 << 31) - 2048, 4096), ((1 << 32) - 2048, 2048 + 77)]
    for i, (at, m) in enumerate(spots):
        x[at:at + m] = gradient(m, i, torch.bfloat16).cuda()
    pay = mx.quantize(x)
    out = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    mx.dequantize(out, pay)
    check_windows(x, lambda at, m: x[at:at + m].float().cpu().numpy(), spots, pay, out, n)
    assert int(out.count_nonzero()) <= sum(m for _, m in spots)
    # the payload of a payload's values is that payload
    again = torch.full_like(pay, 0xa5)
    mx.requantize_n(again, [pay], n)
    assert torch.equal(again, pay)


@gpu
def test_feedback_over_several_launches():
    """float32 with feedback, longer than one launch takes (2^29 elements)."""
    n = (1 << 29) + 1055
    x = torch.zeros(n, device="cuda")
    r = torch.zeros(n, device="cuda")
    spots = [(0, 2048), ((1 << 29) - 1024, 2048 + 31)]
    for i, (at, m) in enumerate(spots):
        x[at:at + m] = gradient(m, i).cuda()
        r[at:at + m] = gradient(m, 9 + i).cuda() * 0.1
    left = torch.full_like(r, 7)
    pay = mx.quantize(x, residual=r, residual_out=left)
    out = torch.empty(n, device="cuda")
    mx.dequantize(out, pay)

    def y(at, m):
        return (x[at:at + m] + r[at:at + m]).cpu().numpy()
    check_windows(x, y, spots, pay, out, n)
    assert torch.equal(left, (x + r) - out)


# ---- with the rest of the framework ------------------------------------------

def fold_of_another_process(inbox, results):
    """A rank that folds what lies in its peer's memory."""
    try:
        pay, n = inbox.get(timeout=60)
        out = torch.empty(n, device="cuda")
        gloo_amd.errors.check(_lib.lib.glx_mx_reduce_n(
            5, out.data_ptr(), P16(pay.data_ptr(), pay.data_ptr()), 2, n, 0.5, None))
        torch.cuda.synchronize()
        hop = torch.empty_like(pay)
        gloo_amd.errors.check(_lib.lib.glx_mx_requantize_n(
            hop.data_ptr(), P16(pay.data_ptr()), 1, n, 1.0, None))
        torch.cuda.synchronize()
        del pay
        results.put((out.cpu().numpy(), hop.cpu().numpy()))
    except BaseException as e:  # noqa: BLE001
        results.put(repr(e))


@gpu
def test_payload_in_another_process():
    """The C ABI takes memory that another process shares: kernels reach it."""
    n = 4099
    ctx = torch.multiprocessing.get_context("spawn")
    inbox, results = ctx.Queue(), ctx.Queue()
    child = ctx.Process(target=fold_of_another_process, args=(inbox, results))
    child.start()
    x = gradient(n, 4)
    pay = mx.quantize(x.cuda())
    torch.cuda.synchronize()
    inbox.put((pay, n))
    got = results.get(timeout=100)
    child.join(30)
    assert not isinstance(got, str), got
    exp, values = payload_of(x.numpy())
    same_bits(got[0], values.astype(np.float32))
    assert np.array_equal(got[1][:exp.size], exp)


@gpu
def test_compressed_exchange_of_ranks():
    """Four thread-ranks squeeze their gradients with feedback, send the payloads
    to each other with the copy kernel, fold them into the mean and clip it: the
    same bits on every rank, those of the restatement."""
    P, n, steps = 4, 30011, 3
    grads = [[gradient(n, 10 * r + s) for s in range(steps)] for r in range(P)]
    size = mx.payload_bytes(n)
    inbox = [torch.zeros(P, size, dtype=torch.uint8, device="cuda") for _ in range(P)]
    torch.cuda.synchronize()
    gate = threading.Barrier(P)
    results, errs = [[] for _ in range(P)], []

    def rank(r):
        try:
            torch.cuda.set_device(0)
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                err = torch.zeros(n, device="cuda")
                mean = torch.empty(n, device="cuda")
                norm = gloo_amd.Gradients([mean[:n // 2], mean[n // 2:]])
                for step in range(steps):
                    pay = mx.quantize(grads[r][step].cuda(), residual=err, residual_out=err)
                    for q in range(P):
                        gloo_amd.kernel_copy(inbox[q][r].data_ptr(), pay.data_ptr(), size, 8, s)
                    s.synchronize()
                    gate.wait(60)
                    mx.reduce_n(mean, list(inbox[r]), scale=1.0 / P)
                    total = norm.clip_norm(1.0)
                    s.synchronize()
                    results[r].append((mean.cpu().numpy(), float(total)))
                    gate.wait(60)
        except BaseException as e:  # noqa: BLE001
            errs.append(e)
            gate.abort()

    ts = [threading.Thread(target=rank, args=(r,)) for r in range(P)]
    [t.start() for t in ts]
    [t.join(120) for t in ts]
    assert not errs, errs
    err = [np.zeros(n, np.float32) for _ in range(P)]
    for step in range(steps):
        pays = []
        for r in range(P):
            y = grads[r][step].numpy() + err[r]
            p, v = payload_of(y)
            err[r] = (y - v).astype(np.float32)
            pays.append(p)
        mean = fold_of(pays, n, 1.0 / P).astype(np.float64)
        total = np.sqrt((mean ** 2).sum())
        exp = mean * min(1.0, 1.0 / (total + 1e-6))
        for r in range(P):
            got, norm = results[r][step]
            assert np.array_equal(got, results[0][step][0])
            assert abs(norm - total) <= 2.0 ** -24 * total * (1 + 1e-6)
            # the coefficient and the product are rounded to fp32 once each
            assert np.all(np.abs(got - exp) <= 2.0 ** -23 * 1.001 * np.abs(exp) + 2.0 ** -149)
