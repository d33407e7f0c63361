"""The teacher / student operators (functional.quantize_rows, linear_int8, top_logits, distill_loss) against plain implementations in
64 bits, their refusals, and a run of them together.

Tolerances count roundings: u = 2^-24 for fp32, half a step (finfo.eps / 2) for a result stored in fewer bits."""
import ctypes
import math

import numpy as np
import pytest
import torch

from subreg_hip import _lib, functional as HF

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda t: str(t).replace("torch.", "")  # noqa: E731


def rnd(shape, seed, dtype=torch.float32, scale=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(device)


def stored(t):
    """Half a step of a stored value, and half the smallest subnormal."""
    f = torch.finfo(t)
    return f.eps / 2, f.smallest_normal * f.eps / 2


# ------------------------------------------------------------------------------------------------ plain forms, 64 bits
def plain_codes(x):
    """(codes, scale) of rows: quotients and product rounded to fp32 once (a double holds each exactly enough to round once)."""
    x = x.detach().cpu().double().numpy()
    bad = ~np.isfinite(x).all(1)
    amax = np.maximum(np.abs(np.where(np.isfinite(x), x, 0.0)).max(1), 2.0 ** -100)
    inv = (127.0 / amax).astype(np.float32).astype(np.float64)
    scale = (amax / 127.0).astype(np.float32)
    prod = (np.where(np.isfinite(x), x, 0.0) * inv[:, None]).astype(np.float32).astype(np.float64)
    codes = np.clip(np.rint(prod), -127, 127).astype(np.int8)
    codes[bad] = 0
    scale[bad] = np.nan
    return codes, scale


def plain_linear(codes, scale, w, ws, bias):
    """(y, |product|) in 64 bits."""
    prod = (codes.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64) * scale.astype(np.float64)[:, None] * ws.astype(np.float64)
    return (prod if bias is None else prod + bias.astype(np.float64)), np.abs(prod)


def plain_top(z, k):
    z = z.detach().cpu().double()
    key = torch.where(torch.isnan(z), torch.tensor(math.inf), z)
    order = torch.tensor(np.lexsort((np.broadcast_to(np.arange(z.shape[1]), z.shape), -key.numpy(), ~torch.isnan(z).numpy()), axis=1))[:, :k]
    return z.gather(1, order), order


def plain_distill(z, tv, ti, y, temp=1.0, kd=1.0, ce=0.0, ignore=-100, reduction="mean"):
    """(loss, gradient for g = 1, rows' losses, per-row gradients of the 'none' form) in 64 bits."""
    z, tv, ti = z.detach().cpu().double(), tv.detach().cpu().double(), ti.cpu().long()
    n, v = z.shape
    keep = (ti >= 0) & (tv != -math.inf)
    has_kd = keep.any(1)
    has_ce = torch.zeros(n, dtype=torch.bool) if y is None or ce == 0 else y.cpu() != ignore
    kls, ces, gk, gc = torch.zeros(n).double(), torch.zeros(n).double(), torch.zeros(n, v).double(), torch.zeros(n, v).double()
    for r in range(n):
        if has_kd[r]:
            i, t = ti[r][keep[r]], tv[r][keep[r]] / temp
            if (i >= v).any():
                kls[r], gk[r] = math.nan, math.nan
            else:
                p = torch.softmax(t, 0)
                logq = torch.log_softmax(z[r] / temp, 0)
                live = p > 0
                kls[r] = (p[live] * (torch.log_softmax(t, 0)[live] - logq[i][live])).sum()
                gk[r] = (torch.softmax(z[r] / temp, 0).index_add(0, i, -p)) / temp
        if has_ce[r]:
            lab = int(y[r])
            if not 0 <= lab < v:
                ces[r], gc[r] = math.nan, math.nan
            else:
                ces[r] = -torch.log_softmax(z[r], 0)[lab]
                gc[r] = torch.softmax(z[r], 0)
                gc[r, lab] -= 1
    wk, wc = kd * temp * temp, ce
    if reduction == "mean":
        nk, nc = max(1, int(has_kd.sum())), max(1, int(has_ce.sum()))
        return wk * kls.sum() / nk + wc * ces.sum() / nc, wk / nk * gk + wc / nc * gc
    if reduction == "sum":
        return wk * kls.sum() + wc * ces.sum(), wk * gk + wc * gc
    return wk * kls + wc * ces, wk * gk + wc * gc


def distill_bounds(z, tv, ti, temp, kd, ce):
    """(error of one row's loss, error of a gradient element before it is stored).

    With x = (m - z_v) / T an exp carries (3 x + 3) u (subtraction, constant, product, 1 ulp of the exponential), a softmax sum the
    mean of that under q, where sum q x <= ln V, and the additions (log2 V + V / 256 a thread) u; the same for the teacher's side.
    A loss term adds the exponents' own roundings, 3 u x at the kept entries and the label.  A gradient element is a difference of
    probabilities <= 1, each with the relative error of its exp (x e^-x <= 1/e) and of the sum."""
    z = z.detach().cpu().double()
    z = torch.where(torch.isfinite(z), z, z[torch.isfinite(z)].min() if torch.isfinite(z).any() else torch.tensor(0.0).double())
    v = z.shape[1]
    spread = float((z.max(1).values - z.min(1).values).max())
    t = tv.detach().cpu().double()
    t = t[torch.isfinite(t)]
    tspread = float(t.max() - t.min()) if t.numel() else 0.0
    sums = 3 * math.log(v) + 3 + math.log2(v) + v / 256 + 3 * math.log(256) + 3 + 8
    row = U * ((sums + 4 * (spread + tspread) / temp + 16) * abs(kd) * temp * temp + (sums + 4 * spread + 16) * abs(ce))
    elem = U * (2 * sums + 8) * (abs(kd) * temp + abs(ce))
    return row, elem


def close(got, want, bound, dtype=torch.float32, note=""):
    got, want = got.detach().cpu().double(), want.double()
    rel, low = stored(dtype)
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), note
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), note
    if torch.is_tensor(bound) and bound.dim():
        bound = bound.expand(want.shape)[fin]
    err = (got - want).abs()[fin]
    tol = (bound + want.abs()[fin] * rel * 1.001 + low)
    assert bool((err <= tol).all()), "%s: error %.3g, allowed %.3g" % (note, float((err - tol).max()), float(tol.max()))


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
def test_refusals_on_cpu():
    f = torch.zeros
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        HF.quantize_rows(f(2, 8))
    with pytest.raises(TypeError):
        HF.quantize_rows(f(2, 8, dtype=torch.float64))
    with pytest.raises(ValueError):
        HF.quantize_rows(f(2, 0))
    w, s = f(5, 8, dtype=torch.int8), f(5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        HF.linear_int8(f(2, 8), w, s)
    for bad in (dict(weight=f(5, 8)), dict(weight=f(5, 9, dtype=torch.int8)), dict(weight_scale=f(4)), dict(weight_scale=s.double()),
                dict(bias=f(4)), dict(bias=s.half()), dict(x_scale=f(2)), dict(x=f(2, 8, dtype=torch.int8)),
                dict(x=f(2, 8, dtype=torch.int8), x_scale=f(3)), dict(weight=f(0, 8, dtype=torch.int8), weight_scale=f(0))):
        with pytest.raises(ValueError):
            HF.linear_int8(**{**dict(x=f(2, 8), weight=w, weight_scale=s), **bad})
    for bad in (dict(x=f(2, 8, dtype=torch.float64)), dict(out_dtype=torch.float64), dict(x=f(2, 8, dtype=torch.int32))):
        with pytest.raises(TypeError):
            HF.linear_int8(**{**dict(x=f(2, 8), weight=w, weight_scale=s), **bad})
    with pytest.raises(ValueError, match="exact"):
        k = _lib.I8_MAX_DIM + 1
        HF.linear_int8(f(1, k), f(1, k, dtype=torch.int8), f(1))
    with pytest.raises(RuntimeError, match="no gradient"):
        HF.linear_int8(f(2, 8, requires_grad=True), w, s)
    for k in (0, 9, -1):
        with pytest.raises(ValueError):
            HF.top_logits(f(2, 8), k)
    with pytest.raises(ValueError):
        HF.top_logits(f(2, 400), 257)
    with pytest.raises(TypeError):
        HF.top_logits(f(2, 8, dtype=torch.int32), 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        HF.top_logits(f(2, 8), 1)
    many = f(1, 8).expand(1 << 22, 8)
    for call in (lambda: HF.quantize_rows(many), lambda: HF.top_logits(many, 1), lambda: HF.linear_int8(many, w, s),
                 lambda: HF.linear_int8(f(1, 8), w[:1].expand(1 << 22, 8), s[:1].expand(1 << 22))):
        with pytest.raises(ValueError, match="rows"):
            call()
    i = f(2, 3, dtype=torch.int64)
    good = dict(logits=f(2, 8), top_values=f(2, 3), top_indices=i)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        HF.distill_loss(**good)
    for bad in (dict(top_values=f(2, 2)), dict(top_values=f(3, 3), top_indices=f(3, 3, dtype=torch.int64)), dict(target=f(3, dtype=torch.int64)),
                dict(reduction="avg"), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
                dict(kd_weight=math.inf), dict(ce_weight=math.nan), dict(top_values=f(2, 0), top_indices=f(2, 0, dtype=torch.int64)),
                dict(top_values=f(2, 257), top_indices=f(2, 257, dtype=torch.int64)), dict(logits=f(2, 0))):
        with pytest.raises(ValueError):
            HF.distill_loss(**{**good, **bad})
    for bad in (dict(top_indices=f(2, 3)), dict(target=f(2)), dict(logits=f(2, 8, dtype=torch.float64))):
        with pytest.raises(TypeError):
            HF.distill_loss(**{**good, **bad})


def test_c_entries_refuse_on_cpu():
    lib = _lib.load()
    p = 1 << 20                                                     # an aligned address; nothing is launched
    assert lib.subreg_quantize_rows(None, 8, 0, 1, 8, p, 16, p, None) == -1
    assert lib.subreg_quantize_rows(p, 8, 0, 1, 8, p, 7, p, None) == -1
    assert lib.subreg_quantize_rows(p, 8, 3, 1, 8, p, 16, p, None) == -1
    assert lib.subreg_quantize_rows(p, 8, 0, 1 << 22, 8, p, 16, p, None) == -1
    n = lib.subreg_linear_int8_ws_bytes(4, 100, 7, 0, p, 100)
    assert n >= 4 * 100 and lib.subreg_linear_int8_ws_bytes(4, _lib.I8_MAX_DIM + 1, 7, 0, p, 100) == -1
    args = [p, 100, 0, None, p, 100, p, None, p, 0, 4, 100, 7, p, n, None]
    for at, value in ((0, None), (2, 3), (2, 9), (3, p), (9, 3), (10, 0), (11, 0), (11, _lib.I8_MAX_DIM + 1), (12, 0), (12, 1 << 22), (10, 1 << 22), (13, None), (13, p + 8),
                      (14, n - 1), (5, -1)):
        bad = list(args)
        bad[at] = value
        assert lib.subreg_linear_int8(*bad) == -1, at
    for bad in ((None, 8, 0, 1, 8, 1, p, p, None), (p, 8, 0, 1, 8, 9, p, p, None), (p, 300, 0, 1, 300, 257, p, p, None),
                (p, 8, 3, 1, 8, 1, p, p, None), (p, -1, 0, 1, 8, 1, p, p, None), (p, 8, 0, 0, 8, 1, p, p, None),
                (p, 8, 0, 1, (1 << 30) + 1, 1, p, p, None), (p, 8, 0, 1 << 22, 8, 1, p, p, None)):
        assert lib.subreg_top_logits(*bad) == -1
    assert lib.subreg_distill_ws_bytes(0) == -1

    def desc(**kw):
        d = _lib.DistillDesc()
        base = dict(logits=p, top_values=p, top_indices=p, target=None, logits_stride=8, values_stride=3, indices_stride=3, dtype=0,
                    values_dtype=0, rows=2, vocab=8, top=3, temperature=1.0, kd_weight=1.0, ce_weight=0.0, ignore_index=-100,
                    reduction=2, flags=0, loss=p, ws=p, ws_bytes=lib.subreg_distill_ws_bytes(2))
        for k, v in {**base, **kw}.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    for bad in (dict(logits=None), dict(top_values=None), dict(top_indices=None), dict(loss=None), dict(rows=0), dict(rows=1 << 22), dict(vocab=0), dict(top=0),
                dict(top=257), dict(temperature=0.0), dict(temperature=math.nan), dict(dtype=3), dict(values_dtype=3), dict(reduction=3),
                dict(ws=None), dict(ws=p + 4), dict(ws_bytes=8), dict(flags=1), dict(logits_stride=-1)):
        assert lib.subreg_distill_loss(desc(**bad), None) == -1, bad


# ------------------------------------------------------------------------------------------------ quantize_rows, linear_int8
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 640), (2, 4097), (130, 257)])
def test_quantize_rows(rows, dim, dtype):
    x = rnd((rows, dim), 1, dtype, 3.0)
    if rows > 2:
        x[0] = 0                                                    # an empty row
        x[1, dim // 2] = math.inf
        x[2, 0] = math.nan
    q, s = HF.quantize_rows(x)
    qw, sw = plain_codes(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (rows,)
    assert np.array_equal(q.cpu().numpy(), qw)
    assert np.array_equal(s.cpu().numpy(), sw, equal_nan=True)


@gpu
def test_quantize_rows_extremes_and_shapes():
    x = torch.tensor([[1e-44, -1e-45, 0.0], [3e38, -3e38, 1.0], [2.0 ** -100, 2.0 ** -101, 0.0], [-5.0, 5.0, 2.5]]).cuda()
    q, s = HF.quantize_rows(x)
    qw, sw = plain_codes(x)
    assert np.array_equal(q.cpu().numpy(), qw) and np.array_equal(s.cpu().numpy(), sw)
    assert HF.quantize_rows(x[0])[0].shape == (3,) and HF.quantize_rows(x[0])[1].shape == ()
    y = rnd((2, 3, 50), 2)
    q3, s3 = HF.quantize_rows(y.transpose(1, 2))                     # last dimension not contiguous
    qw, sw = plain_codes(y.transpose(1, 2).reshape(-1, 3))
    assert q3.shape == (2, 50, 3) and np.array_equal(q3.reshape(-1, 3).cpu().numpy(), qw) and np.array_equal(s3.reshape(-1).cpu().numpy(), sw)
    assert HF.quantize_rows(torch.zeros(0, 5).cuda())[0].shape == (0, 5)


LINEAR = [(1, 1, 1), (1, 640, 351), (2, 64, 16), (3, 4096, 1000), (5, 17, 33), (16, 128, 64), (17, 129, 65), (33, 1111, 130),
          (1, 20, 100), (1, 2047, 700), (1, 5000, 90), (1, 9000, 50), (30, 200, 9000), (40, 300, 17000), (60, 100, 16500),
          (48, 2048, 257), (64, 640, 351), (100, 96, 700), (129, 512, 129), (257, 384, 300), (300, 1000, 520), (520, 272, 1030),
          (1100, 200, 2100), (2100, 130, 2050), (2600, 65, 5200)]


def check_linear(x, w, ws, bias, got, out_dtype, codes=None):
    qc, qs = codes if codes is not None else plain_codes(x)
    want, prod = plain_linear(qc, qs, w.cpu().numpy(), ws.cpu().numpy(), None if bias is None else bias.cpu().numpy())
    # sum to fp32, two scales, the bias: one rounding each
    bound = torch.tensor(U * (3 * prod + np.abs(want)))
    close(got, torch.tensor(want), bound, out_dtype, "linear")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_int8(m, k, n, dtype):
    x, wf = rnd((m, k), m + k, dtype), rnd((n, k), n, scale=k ** -0.5)
    w, ws = HF.quantize_rows(wf)
    bias = rnd((n,), 5) if (m + n) % 2 else None
    if m > 4:
        x[1], x[3, k // 2], x[4, 0] = 0, math.nan, -math.inf         # an empty row, two rows that are not finite
    got = HF.linear_int8(x, w, ws, bias)
    assert got.dtype == dtype and got.shape == (m, n)
    check_linear(x, w, ws, bias, got, dtype)
    plain = w.contiguous()                                           # rows of odd pitch: they start at any byte
    assert torch.equal(HF.linear_int8(x, plain, ws, bias).nan_to_num(7), got.nan_to_num(7))


@gpu
@pytest.mark.parametrize("m,k,n", [(1, 33, 40), (4, 640, 60), (40, 100, 130), (300, 256, 260), (7, 2000, 300)])
@pytest.mark.parametrize("out_dtype", TYPES, ids=ids)
def test_linear_int8_codes_given(m, k, n, out_dtype):
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    xs, ws = torch.rand(m, generator=g) * 1e-3, torch.rand(n, generator=g) * 1e-3
    got = HF.linear_int8(x.cuda(), w.cuda(), ws.cuda(), None, xs.cuda(), out_dtype)
    check_linear(None, w, ws, None, got, out_dtype, (x.numpy(), xs.numpy()))
    buf = torch.full((m, k + 13), 77, dtype=torch.int8).cuda()       # rows inside a wider buffer, whose other bytes mean nothing
    buf[:, 5:5 + k] = x.cuda()
    assert torch.equal(HF.linear_int8(buf[:, 5:5 + k], w.cuda(), ws.cuda(), None, xs.cuda(), out_dtype), got)


@gpu
def test_linear_int8_largest_sums_are_exact():
    for k in (131071, 65536):
        x = torch.full((2, k), -128, dtype=torch.int8).cuda()
        w = torch.full((3, k), -128, dtype=torch.int8).cuda()
        w[1] = 127
        one = torch.ones(3).cuda()
        got = HF.linear_int8(x, w, one, None, one[:2])
        want = torch.tensor([128.0 * 128 * k, -128.0 * 127 * k, 128.0 * 128 * k], dtype=torch.float64).float()
        assert torch.equal(got.cpu(), want.expand(2, 3))


# The loops of every kernel at work: tiles of each size with three and more stages of K (whole and ragged edges, out a multiple of 4 or
# not), one row with more channels than the grid has waves for (each length of the row in registers), few rows with more groups of
# channels than the grid has blocks (each number of row tiles), and short rows of many channels, which go to the tiles.
STEADY = [(4096, 512, 3584), (4000, 521, 3601), (3990, 1153, 3600), (2304, 640, 2048), (2250, 777, 2101), (1024, 640, 2048),
          (1000, 650, 2049), (300, 1000, 521), (1, 1000, 40000), (1, 2047, 33001), (1, 4096, 20000), (1, 8192, 9001),
          (5, 2100, 70001), (20, 2048, 66000), (40, 2176, 66001), (64, 2100, 65999), (64, 1024, 32768), (9, 1500, 20003)]


@gpu
@pytest.mark.parametrize("m,k,n", STEADY)
def test_linear_int8_steady_state_is_exact(m, k, n):
    """Codes given and scales of 1: every product is the integer sum, rounded to fp32 once (64-bit floats hold the sums exactly)."""
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device="cuda")
    pitch = (k + 15) // 16 * 16                                      # rows as quantize_rows lays them out: read by the tiles as they are
    w = torch.randint(-128, 128, (n, pitch), generator=g, dtype=torch.int8, device="cuda")[:, :k]
    got = HF.linear_int8(x, w, torch.ones(n, device="cuda"), None, torch.ones(m, device="cuda"))
    for lo in range(0, n, 8192):
        want = x.double() @ w[lo:lo + 8192].double().t().contiguous()
        assert torch.equal(got[:, lo:lo + 8192], want.float()), lo


@gpu
def test_linear_int8_codes_past_one_pass_of_the_grid():
    """More than 2^30 bytes of codes (2^26 threads' worth): rows at both ends and at the grid's turn are those of a call on them alone."""
    m, k, n = 8500, 131071, 3
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device="cuda")
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8, device="cuda")
    one = torch.ones(m, device="cuda")
    got = HF.linear_int8(x, w, one[:n], None, one)
    for rows in (slice(0, 40), slice(8180, 8220), slice(m - 40, m)):
        want = x[rows].double() @ w.double().t().contiguous()
        assert torch.equal(got[rows], want.float())


@gpu
def test_linear_int8_strides_and_leading_dimensions():
    x, wf = rnd((4, 6, 200), 1), rnd((90, 200), 2)
    w, ws = HF.quantize_rows(wf)
    base = HF.linear_int8(x.reshape(24, 200), w, ws)
    assert torch.equal(HF.linear_int8(x, w, ws).reshape(24, 90), base)
    wide = torch.full((24, 333), 9.0).cuda()
    wide[:, 100:300] = x.reshape(24, 200)
    assert torch.equal(HF.linear_int8(wide[:, 100:300], w, ws), base)
    assert torch.equal(HF.linear_int8(x.transpose(0, 1), w, ws), base.view(4, 6, 90).transpose(0, 1))
    assert torch.equal(HF.linear_int8(x[0, 0], w, ws), base[0])
    assert torch.equal(HF.linear_int8(x[:1, 0].expand(5, 200), w, ws), base[:1].expand(5, 90))      # one row seen many times
    assert HF.linear_int8(x[:0], w, ws).shape == (0, 6, 90)
    last = torch.zeros(89 * 208 + 200, dtype=torch.int8).cuda().as_strided((90, 200), (208, 1))     # the last row ends with the storage
    last.copy_(w)
    assert torch.equal(HF.linear_int8(x, last, ws).reshape(24, 90), base)


# ------------------------------------------------------------------------------------------------ top_logits
def check_top(z, k):
    values, indices = HF.top_logits(z, k)
    wv, wi = plain_top(z.reshape(-1, z.shape[-1]), k)
    assert values.dtype == z.dtype and indices.dtype == torch.int64 and values.shape == z.shape[:-1] + (k,)
    assert torch.equal(indices.reshape(-1, k).cpu(), wi)
    assert torch.equal(values.reshape(-1, k).cpu().double().nan_to_num(1e9), wv.nan_to_num(1e9))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (64, 351, 5), (5, 60, 60), (2, 256, 256), (7, 1000, 17), (3, 1025, 256),
                                          (2, 5003, 64), (9, 32000, 32), (1, 16384, 256), (1, 16385, 1), (3, 131071, 256), (60, 20011, 40), (300, 33333, 50), (1, 131072, 128), (2, 140001, 256), (1, 300007, 33)])
def test_top_logits(rows, vocab, k, dtype):
    check_top(rnd((rows, vocab), vocab + k, dtype, 2.5), k)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("vocab,k", [(37, 9), (1000, 256), (4099, 200), (70000, 100)])
def test_top_logits_ties_masks_and_nan(vocab, k, dtype):
    z = rnd((14, vocab), 3, dtype)
    low = torch.finfo(dtype).min
    z[0] = 0                                                         # all equal
    z[1] = -math.inf                                                 # a mask that leaves nothing
    z[2] = low
    z[3, k // 2:] = -math.inf                                        # fewer numbers than k
    z[4, ::2] = math.inf
    z[5, 3] = math.nan
    z[6] = math.nan
    z[7, ::3], z[7, 1::3] = 0.0, -0.0                                # +0 = -0
    z[8] = z[8].round()                                              # many ties at the border
    z[9] = 1.0
    z[9, -1] = 2.0
    z[10] = torch.arange(vocab).cuda().to(dtype).clamp(max=60000)
    z[11] = -torch.arange(vocab).cuda().to(dtype).clamp(max=60000)
    z[12, : vocab // 2] = low
    z[13] = -math.inf
    z[13, -1] = math.nan
    check_top(z, k)


@gpu
def test_top_logits_strides_and_leading_dimensions():
    z = rnd((3, 4, 777), 4)
    check_top(z, 20)
    wide = rnd((12, 1001), 5, torch.bfloat16)
    for lo in (0, 1, 3):
        check_top(wide[:, lo:lo + 777], 20)
    check_top(z.transpose(0, 1), 7)
    check_top(z[0, :1].expand(5, 777), 3)
    check_top(z[0, 0], 3)
    v, i = HF.top_logits(z[:0], 4)
    assert v.shape == (0, 4, 4) and i.shape == (0, 4, 4)


# ------------------------------------------------------------------------------------------------ distill_loss
def make_distill(n, v, k, dtype, seed, labels=True, scale=2.5):
    z = rnd((n, v), seed, dtype, scale)
    tv, ti = torch.topk(0.7 * z.float() + rnd((n, v), seed + 1, scale=2.0), k, dim=1)
    kept = torch.randint(1, k + 1, (n, 1), generator=torch.Generator().manual_seed(seed)).cuda()
    ti = ti.masked_fill(torch.arange(k).cuda()[None] >= kept, -1)
    y = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(seed + 2)).cuda() if labels else None
    return z, tv.to(dtype), ti, y


def check_distill(z, tv, ti, y, temp=1.0, kd=1.0, ce=0.0, reduction="mean", g=None, ignore=-100):
    leaf = z.detach().requires_grad_()
    loss = HF.distill_loss(leaf, tv, ti, y, temp, kd, ce, ignore, reduction)
    flat = z.reshape(-1, z.shape[-1])
    k = tv.shape[-1]
    want, grad = plain_distill(flat, tv.reshape(-1, k), ti.reshape(-1, k), None if y is None else y.reshape(-1), temp, kd, ce, ignore, reduction)
    row, elem = distill_bounds(flat, tv, ti, temp, kd, ce)
    n = flat.shape[0]
    assert loss.dtype == torch.float32
    close(loss.reshape(-1), want.reshape(-1), row * (n if reduction == "sum" else 2), note="loss")     # (mean: two terms' means)
    if g is None:
        (loss.sum() if reduction == "none" else loss).backward()
    else:
        loss.backward(g)
        gg = g.detach().cpu().double()
        grad = grad * (gg.reshape(-1, 1) if reduction == "none" else gg)
        elem = elem * float(gg.abs().max())
    assert leaf.grad.dtype == z.dtype and leaf.grad.shape == z.shape
    close(leaf.grad.reshape(-1, z.shape[-1]), grad, elem, z.dtype, "gradient")
    with torch.no_grad():                                            # the loss alone: sums in another order, the same bound
        alone = HF.distill_loss(leaf, tv, ti, y, temp, kd, ce, ignore, reduction)
    close(alone.reshape(-1), want.reshape(-1), row * (n if reduction == "sum" else 2), note="the loss alone")
    return loss.detach(), leaf.grad


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n,v,k,temp", [(1, 1, 1, 1.0), (2, 3, 2, 2.0), (64, 60, 10, 4.0), (5, 351, 256, 1.0), (3, 1000, 7, 2.0),
                                        (70, 1537, 64, 3.0), (4, 5003, 33, 0.5), (2, 32000, 64, 2.0), (130, 2048, 50, 1.0),
                                        (1, 131072, 128, 2.0), (2, 140003, 20, 1.5)])
def test_distill_loss(n, v, k, temp, dtype):
    z, tv, ti, y = make_distill(n, v, k, dtype, n + v)
    if n > 4:
        ti[1] = -1                                                   # no entries, but a label
        y[2] = -100                                                  # entries, no label
        ti[3], y[3] = -1, -100                                       # neither
        z[3] = math.nan                                              # ... whatever its logits hold
    check_distill(z, tv, ti, y, temp, 1.0, 0.0)
    check_distill(z, tv, ti, y, temp, 0.7, 0.4)
    check_distill(z, tv, ti, y, temp, 0.7, 0.4, "sum")
    check_distill(z, tv, ti, y, temp, 0.7, 0.4, "none")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("v", [61, 4100])
def test_distill_upstream_factors(v, dtype):
    z, tv, ti, y = make_distill(9, v, 8, dtype, 4)
    for reduction in ("mean", "sum"):
        for g in (1.0, 0.25, -3.0, 0.0, 1024.0):
            check_distill(z, tv, ti, y, 2.0, 0.5, 0.5, reduction, torch.tensor(g).cuda())
    g = torch.tensor([1.0, 0.0, -2.0, 1.0, 0.5, 3.0, 1.0, 100.0, 1.0]).cuda()
    check_distill(z, tv, ti, y, 2.0, 0.5, 0.5, "none", g)
    check_distill(z, tv, ti, y, 2.0, 0.5, 0.5, "none", torch.tensor(2.0).cuda().expand(9))


@gpu
def test_distill_loss_scale_keeps_small_gradients_in_fp16():
    z, tv, ti, y = make_distill(512, 2000, 4, torch.float16, 4)
    _, grad = check_distill(z, tv, ti, y, 1.0, 1.0, 0.0, "mean", torch.tensor(4096.0).cuda())
    assert float((grad == 0).float().mean()) < 0.01                  # (unscaled, most of them are below fp16's smallest number)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("v", [40, 3001])
def test_distill_masks_and_bad_entries(v, dtype):
    low = torch.finfo(dtype).min
    z, tv, ti, y = make_distill(12, v, 6, dtype, 5)
    ti = torch.topk(z.float(), 6, dim=1).indices
    tv[0, 2:] = -math.inf                                            # masked by value
    tv[1] = -math.inf                                                # all of them
    ti[2] = torch.tensor([5, 5, 5, 7, 7, 5]).cuda()                  # the same index many times
    y[2] = 5
    ti[3, 1] = v                                                     # out of range
    y[4] = v
    y[5] = -1
    z[6, 10:] = -math.inf                                            # masked logits, none of them kept
    ti[6], y[6] = torch.tensor([0, 1, 2, 3, 4, 5]).cuda(), 9
    z[7, 10:] = low
    ti[7], y[7] = torch.tensor([0, 1, 2, 3, 4, 5]).cuda(), 0
    tv[8, 1:] = low                                                  # shares that vanish
    z[9] = low                                                       # all at the lowest number: a uniform row
    ti[10], y[10] = -1, -100
    z[10] = math.inf
    ti[11], tv[11] = torch.tensor([-5, -1, 2, -1, 3, -1]).cuda(), torch.tensor([9.0, 8.0, 1.0, 50.0, 1.0, 4.0]).cuda().to(dtype)
    rows, grad = check_distill(z, tv, ti, y, 2.0, 1.0, 0.5, "none")
    bad = torch.isnan(rows).cpu()
    assert bad.tolist() == [i in (3, 4, 5) for i in range(12)]
    assert torch.isnan(grad).all(1).cpu().tolist() == bad.tolist() and float(grad[10].abs().sum()) == 0.0
    ok = ~bad
    check_distill(z[ok], tv[ok], ti[ok], y[ok], 2.0, 1.0, 0.5, "mean")
    # a logit of -inf where the teacher has a share: the loss is infinite, the gradient is not
    z[0, ti[0, 0]] = -math.inf
    leaf = z[:1].detach().requires_grad_()
    loss = HF.distill_loss(leaf, tv[:1], ti[:1], None, 2.0)
    loss.backward()
    assert loss.item() == math.inf and torch.isfinite(leaf.grad).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("v", [300, 3001, 50021, 140003])
@pytest.mark.parametrize("temp", [1.0, 2.0, 3.0, 0.01])
def test_distill_numbers_as_masks_and_far_logits(v, dtype, temp):
    """Masks that are large numbers, in part of a row (whole threads see nothing else) and in all of it; logits far from 0."""
    masks = [-1e4, -1e6, -3e7, -1e9, -1e10, -1e20, -1e30, torch.finfo(dtype).min]
    z = rnd((2 * len(masks) + 6, v), 3, dtype, 2.5)
    for i, m in enumerate(masks):
        z[2 * i, 40:] = m
        z[2 * i + 1] = m
    for i, far in enumerate((1e4, -1e4, 1e6, -1e6, 1e8, -1e8)):
        z[2 * len(masks) + i] = (z[2 * len(masks) + i].float() + far).to(dtype)
    n = z.shape[0]
    ti = torch.arange(30, 38).expand(n, 8).clone().cuda()
    tv = rnd((n, 8), 4, dtype)
    y = torch.arange(n).cuda()
    near = torch.where(z < z.max(1, keepdim=True).values - 200, z.max(1, keepdim=True).values, z)    # (masked logits carry no share)
    row, elem = distill_bounds(near, tv, ti, temp, 0.5, 0.5)
    for reduction in ("none", "mean"):
        leaf = z.detach().requires_grad_()
        loss = HF.distill_loss(leaf, tv, ti, y, temp, 0.5, 0.5, reduction=reduction)
        loss.sum().backward()
        want, grad = plain_distill(z, tv, ti, y, temp, 0.5, 0.5, reduction=reduction)
        close(loss.detach().reshape(-1), want.reshape(-1), 2 * row, note="loss")
        close(leaf.grad, grad, elem, dtype, "gradient")
        with torch.no_grad():
            alone = HF.distill_loss(leaf, tv, ti, y, temp, 0.5, 0.5, reduction=reduction)
        close(alone.reshape(-1), want.reshape(-1), 2 * row, note="the loss alone")


@gpu
@pytest.mark.parametrize("n,v,dtype", [(2100, 32003, torch.bfloat16), (1150, 60000, torch.float16), (530, 131072, torch.bfloat16),
                                       (2100, 16001, torch.float32)])
def test_distill_large_matrices_row_by_row(n, v, dtype):
    """Matrices that go past the caches (128 MB and more): every row's loss and gradient is that of a call on fewer rows, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(n, v, generator=g, device="cuda").mul_(2.5).to(dtype)
    tv, ti = torch.topk(z[:, 7:1000].float(), 30, dim=1)
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[3] = -100
    ti[3] = -1

    def run(rows):
        leaf = z[rows].detach().requires_grad_()
        loss = HF.distill_loss(leaf, tv[rows].to(dtype), ti[rows], y[rows], 2.0, 0.5, 0.5, reduction="none")
        loss.sum().backward()
        return loss.detach(), leaf.grad

    loss, grad = run(slice(0, n))
    for lo in range(0, n, n // 3):
        part = run(slice(lo, lo + n // 3))
        assert torch.equal(part[0], loss[lo:lo + n // 3]) and torch.equal(part[1], grad[lo:lo + n // 3])
    rows = [0, 3, n // 2, n - 1]
    want, wg = plain_distill(z[rows], tv[rows].to(dtype), ti[rows], y[rows], 2.0, 0.5, 0.5, reduction="none")
    row, elem = distill_bounds(z[rows], tv[rows], ti[rows], 2.0, 0.5, 0.5)
    close(loss[rows], want, row)
    close(grad[rows], wg, elem, dtype)


@gpu
def test_distill_strides_types_and_leading_dimensions():
    z, tv, ti, y = make_distill(12, 501, 6, torch.bfloat16, 6)
    base, grad = check_distill(z, tv, ti, y, 2.0, 0.5, 0.5)
    wide = torch.zeros(12, 520, dtype=torch.bfloat16).cuda()
    wide[:, 7:508] = z
    l2, g2 = check_distill(wide[:, 7:508], tv, ti, y, 2.0, 0.5, 0.5)
    assert torch.equal(l2, base) and torch.equal(g2, grad)
    l3, g3 = check_distill(z.view(3, 4, 501), tv.view(3, 4, 6), ti.view(3, 4, 6), y.view(3, 4), 2.0, 0.5, 0.5)
    assert torch.equal(l3, base) and torch.equal(g3.view(12, 501), grad)
    check_distill(z.view(3, 4, 501).transpose(0, 1), tv.view(3, 4, 6).transpose(0, 1), ti.view(3, 4, 6).transpose(0, 1),
                  y.view(3, 4).t(), 2.0, 0.5, 0.5, "none")
    check_distill(z, tv.float(), ti, y, 2.0, 0.5, 0.5)               # the teacher in another type
    check_distill(z, tv, ti, y.int(), 2.0, 0.5, 0.5)
    check_distill(z, tv, ti.int(), y, 2.0, 0.5, 0.5)
    row = z[:1].detach().requires_grad_()                            # one row of logits against twelve teachers: the gradients add
    loss = HF.distill_loss(row.expand(12, 501), tv, ti, y, 2.0, 0.5, 0.5, reduction="sum")
    loss.backward()
    _, want = plain_distill(z[:1].expand(12, 501), tv, ti, y, 2.0, 0.5, 0.5, reduction="sum")
    # twelve rows, each stored in bf16, summed by autograd in bf16 or wider: 12 + 11 half steps of the largest partial sum
    _, elem = distill_bounds(z[:1], tv, ti, 2.0, 0.5, 0.5)
    bound = 12 * elem + 23 * 2.0 ** -8 * want.abs().sum(0)
    close(row.grad[0], want.sum(0), bound, torch.bfloat16, "broadcast rows")
    e = z[:0].detach().requires_grad_()
    loss = HF.distill_loss(e, tv[:0], ti[:0], y[:0])
    loss.backward()
    assert loss.item() == 0.0 and e.grad.shape == (0, 501) and HF.distill_loss(e, tv[:0], ti[:0], reduction="none").shape == (0,)
    with pytest.raises(TypeError):
        HF.distill_loss(z, tv, ti.float())


@gpu
def test_distill_second_backward_and_changed_inputs():
    z, tv, ti, y = make_distill(8, 300, 6, torch.float32, 7)
    leaf = z.detach().requires_grad_()
    loss = HF.distill_loss(leaf, tv, ti, y, 2.0, 0.5, 0.5)
    (a,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    keep = a.clone()
    a.mul_(0)                                                        # the first gradient is the caller's
    (b,) = torch.autograd.grad(3 * loss, leaf, retain_graph=True)
    (c,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(c, keep)
    _, elem = distill_bounds(z, tv, ti, 2.0, 0.5, 0.5)
    close(b, 3 * keep.cpu().double(), 6 * elem)                      # both are within 3 (1) times the bound of the formula's
    inner = z.detach().requires_grad_() * 1.0
    loss = HF.distill_loss(inner, tv, ti, y)
    inner.detach().mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    assert not HF.distill_loss(z, tv, ti, y).requires_grad


def test_distill_temperature_range_on_cpu():
    f = torch.zeros
    good = dict(logits=f(2, 8), top_values=f(2, 3), top_indices=f(2, 3, dtype=torch.int64))
    for bad in (dict(temperature=1e16), dict(temperature=1e-31), dict(temperature=1e12, kd_weight=1e7), dict(kd_weight=1e31)):
        with pytest.raises(ValueError):
            HF.distill_loss(**good, **bad)
    for edge in (dict(temperature=1e15), dict(temperature=1e-30), dict(temperature=1e12, kd_weight=1e5), dict(temperature=0.5, kd_weight=1e30)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            HF.distill_loss(**good, **edge)
    lib, p = _lib.load(), 1 << 20
    for t, kd, ce in ((1e16, 1.0, 0.0), (1e-31, 1.0, 0.0), (math.inf, 1.0, 0.0), (1e12, 1e7, 0.0), (1.0, math.nan, 0.0), (1.0, 1.0, 1e31)):
        d = _lib.DistillDesc(logits=p, top_values=p, top_indices=p, logits_stride=8, values_stride=3, indices_stride=3, rows=2, vocab=8,
                             top=3, temperature=t, kd_weight=kd, ce_weight=ce, reduction=2, loss=p, ws=p, ws_bytes=lib.subreg_distill_ws_bytes(2))
        assert lib.subreg_distill_loss(ctypes.byref(d), None) == -1, (t, kd, ce)


@gpu
@pytest.mark.parametrize("v", [5, 60, 3001, 140003])
@pytest.mark.parametrize("temp", [1e-30, 1e-12, 1e-3, 1e3, 1e10, 1e15])
def test_distill_temperature_range(v, temp):
    """The ends of the accepted range: nothing overflows that the loss itself does not."""
    z, tv, ti, y = make_distill(6, v, 4, torch.float32, 3)
    for reduction in ("none", "sum", "mean"):
        check_distill(z, tv, ti, y, temp, 1.0, 0.5, reduction)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("v", [7, 300, 4100, 50021, 140003])
@pytest.mark.parametrize("temp", [0.25, 1.0, 2.0, 3.0])
def test_distill_kept_entries_and_labels_at_the_lowest_number(v, temp, dtype):
    """A student masked by its type's lowest number where the teacher has a share, or the label is: the loss is that large, not
    infinite."""
    z, _, _, _ = make_distill(3, v, 4, dtype, 6)
    low = torch.finfo(dtype).min
    z[:, 4:] = low
    ti = torch.tensor([[0, 1, 2, 5], [3, 5, 6, 0], [0, 1, 2, 3]]).cuda()
    tv = torch.tensor([[1.0, 0.5, 0.0, -1.0], [2.0, -2.0, -3.0, 1.0], [0.0, 0.0, 0.0, 0.0]]).cuda().to(dtype)
    y = torch.tensor([1, 0, 6]).cuda()
    # (T p < 0.7 for the masked entries, ce = 1/4: every row's loss fits fp32.)  At such numbers a bound is relative: differences,
    # products and sums of at most four shares, each rounded, and the shares' own error, where exponents reach 5 / T
    many = U * (64 + 4 * 5 / temp)
    for kd, ce in ((1.0, 0.0), (0.25, 0.25)):
        leaf = z.detach().requires_grad_()
        loss = HF.distill_loss(leaf, tv, ti, y, temp, kd, ce, reduction="none")
        loss.sum().backward()
        want, grad = plain_distill(z, tv, ti, y, temp, kd, ce, reduction="none")
        assert float(want.max()) > 1 and bool(torch.isfinite(want.float()).all())
        near = torch.where(z == low, z[:, :4].float().min().to(dtype), z)
        row, elem = distill_bounds(near, tv, ti, temp, kd, ce)
        close(loss, want, row + many * want, note="loss")
        close(leaf.grad, grad, elem, dtype, "gradient")
        with torch.no_grad():
            close(HF.distill_loss(leaf, tv, ti, y, temp, kd, ce, reduction="none"), want, row + many * want, note="the loss alone")


@gpu
@pytest.mark.parametrize("temp,kd,ce", [(1.0, 1e30, 0.0), (1.0, 0.0, 1e30), (1e15, 1.0, 0.0), (1e-30, 1e30, 1e30), (1e10, -1e10, 0.0)])
def test_distill_largest_weights(temp, kd, ce):
    """The ends of what the arguments' check accepts are accepted below it, too (1e30 is a little more than 1e30 in fp32)."""
    z, tv, ti, y = make_distill(4, 60, 4, torch.float32, 5)
    for reduction in ("none", "mean"):
        check_distill(z, tv, ti, y, temp, kd, ce, reduction)


@gpu
@pytest.mark.parametrize("v", [60, 3000, 140003])
@pytest.mark.parametrize("reduction", [_lib.REDUCE_SUM, _lib.REDUCE_MEAN])
def test_distill_counted_workspace(v, reduction):
    """The C entry with counts that an earlier gradient call left: the same bits as a call that counts for itself, with the logits' rows
    elsewhere and another factor."""
    lib, n, k = _lib.load(), 300, 9
    z, tv, ti, y = make_distill(n, v, k, torch.float32, 12)
    ti[5], y[7] = -1, -100
    moved = torch.zeros(n, v + 5, device="cuda")
    moved[:, :v] = z
    ws = [torch.empty(lib.subreg_distill_ws_bytes(n), dtype=torch.uint8, device="cuda").fill_(0x5a) for _ in range(2)]
    loss, factor = torch.empty(1, device="cuda"), torch.full((1,), 0.375, device="cuda")

    def call(rows, ws, flags, **out):
        d = _lib.DistillDesc(logits=rows.data_ptr(), top_values=tv.data_ptr(), top_indices=ti.data_ptr(), target=y.data_ptr(),
                             logits_stride=rows.stride(0), values_stride=k, indices_stride=k, dtype=0, values_dtype=0, rows=n, vocab=v,
                             top=k, temperature=2.0, kd_weight=0.5, ce_weight=0.5, ignore_index=-100, reduction=reduction, flags=flags,
                             ws=ws.data_ptr(), ws_bytes=ws.numel(), **{name: t.data_ptr() for name, t in out.items()})
        _lib.check(lib.subreg_distill_loss(ctypes.byref(d), _lib.stream_ptr()), "distill_loss")

    a, b, c = (torch.empty(n, v, device="cuda") for _ in range(3))
    call(z, ws[0], 0, loss=loss, dlogits=a)
    call(moved[:, :v], ws[0], _lib.DISTILL_COUNTED, dlogits=b, grad_scale=factor)
    call(z, ws[1], 0, dlogits=c, grad_scale=factor)
    assert torch.equal(b, c)
    want, grad = plain_distill(z, tv, ti, y, 2.0, 0.5, 0.5, reduction="sum" if reduction == _lib.REDUCE_SUM else "mean")
    row, elem = distill_bounds(z, tv, ti, 2.0, 0.5, 0.5)
    close(loss, want.reshape(1), row * (n if reduction == _lib.REDUCE_SUM else 2), note="loss")
    close(a, grad, elem, note="gradient")
    close(b, 0.375 * grad, 0.375 * elem, note="gradient with a factor")


@gpu
def test_distill_gradient_against_differences():
    z, tv, ti, y = make_distill(6, 77, 5, torch.float32, 8, scale=1.0)
    leaf = z.detach().requires_grad_()
    HF.distill_loss(leaf, tv, ti, y, 2.0, 0.5, 0.5, reduction="sum").backward()
    d = rnd((6, 77), 9)
    h = 2.0 ** -5
    ends = [float(HF.distill_loss(z + s * h * d, tv, ti, y, 2.0, 0.5, 0.5, reduction="sum")) for s in (1, -1)]
    slope = float((leaf.grad.double() * d.double()).sum())
    # third derivative of each row's terms along d: at most 0.5 (T^2 / T^3 + 1) max|d|^3 -> h^2 / 6 of it; the losses' own error over 2 h
    row, _ = distill_bounds(z, tv, ti, 2.0, 0.5, 0.5)
    bound = h * h / 6 * 6 * 0.75 * float(d.abs().max()) ** 3 + 2 * 6 * row / (2 * h)
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= bound


# ------------------------------------------------------------------------------------------------ saved-tensor hooks
def test_distill_backward_reads_the_unpacked_tensors(monkeypatch):
    """What the backward's call points at are the tensors that the unpack hook returned, not the forward's, which may be gone; a hook
    that returns other shapes or types is refused (no kernel runs here: the calls are recorded)."""
    calls = []

    def record(dev, fn, what, ref):
        d = ref._obj
        calls.append((what, (d.logits, d.top_values, d.top_indices, d.target), (d.logits_stride, d.values_stride, d.indices_stride)))

    monkeypatch.setattr(HF, "_launch", record)
    for labels in (True, False):
        z, tv = torch.randn(5, 9).requires_grad_(), torch.randn(5, 3)
        ti, y = torch.randint(0, 9, (5, 3)), torch.randint(0, 9, (5,)) if labels else None
        unpacked = []

        def unpack(t):
            # (rows further apart than the saved ones', and a last dimension that is not contiguous: both have to be followed)
            n = torch.empty(t.shape[0], 2 * t[0].numel() + 1, dtype=t.dtype)[:, :2 * t[0].numel():2].view(t.shape) if t.dim() == 2 else t.clone()
            unpacked.append(n.copy_(t))
            return n

        def far(t):
            n = torch.empty(t.shape[0], t[0].numel() + 4, dtype=t.dtype)[:, :t[0].numel()] if t.dim() == 2 else t.clone()
            unpacked.append(n.copy_(t))
            return n

        args = (2.0, 0.5, 0.5, -100, _lib.REDUCE_MEAN)
        for hook in (lambda t: t, far, unpack):
            calls.clear(), unpacked.clear()
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), hook):
                loss = HF.DistillLossFn.apply(z, tv, ti, y, True, (), *args)
            loss.backward()
            assert [c[0] for c in calls] == ["distill_loss", "distill_loss(bwd)"]
            assert all(a != b for a, b in zip(calls[0][1], calls[1][1]) if a)
            assert (calls[1][1][3] is None) == (not labels)
            if hook is far:
                assert list(calls[1][1][:3 + labels]) == [t.data_ptr() for t in unpacked] and calls[1][2] == (13, 7, 7)
            if hook is unpack:
                assert calls[1][2] == (9, 3, 3)                      # rows with a contiguous last dimension were made of them
        for wrong in (lambda t: t[:-1], lambda t: t.double() if t.dtype == torch.float32 else t.int()):
            calls.clear()
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
                loss = HF.DistillLossFn.apply(z, tv, ti, y, True, (), *args)
            with pytest.raises(RuntimeError, match="unpacked"):
                loss.backward()
            assert len(calls) == 1


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("factor", [1.0, 0.5, -3.0])
@pytest.mark.parametrize("v", [60, 4100])
def test_distill_under_saved_tensor_hooks(v, factor, dtype):
    """Offloaded to the host, checkpointed and packed as copies: the gradient is that of the plain call, bit for bit, with the logits'
    own memory given back and overwritten in between."""
    from torch.utils.checkpoint import checkpoint
    z, tv, ti, y = make_distill(9, v, 8, dtype, 4)

    def loss_of(leaf, tv, ti, y):
        return HF.distill_loss(leaf * 1, tv, ti, y, 2.0, 0.5, 0.5)       # (of a result, which only its saved form keeps)

    leaf = z.detach().requires_grad_()
    (factor * loss_of(leaf, tv, ti, y)).backward()
    want = leaf.grad
    _, plain = plain_distill(z, tv, ti, y, 2.0, 0.5, 0.5)
    _, elem = distill_bounds(z, tv, ti, 2.0, 0.5, 0.5)
    close(want, factor * plain, abs(factor) * elem, dtype, "gradient")

    def clones():
        return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone())

    for kind in ("cpu", "clone", "checkpoint"):
        leaf = z.detach().requires_grad_()
        mine = [t.clone() for t in (tv, ti, y)]
        if kind == "checkpoint":
            loss = checkpoint(loss_of, leaf, *mine, use_reentrant=False)
        else:
            with torch.autograd.graph.save_on_cpu() if kind == "cpu" else clones():
                loss = loss_of(leaf, *mine)
        if kind != "checkpoint":                                     # (a checkpoint keeps its function's arguments)
            del mine
        filler = [torch.full((9, v), 3, dtype=dtype, device="cuda") for _ in range(8)] + [torch.full((9, 8), 1, device="cuda") for _ in range(8)]
        (factor * loss).backward()
        assert torch.equal(leaf.grad, want), kind
        del filler


# ------------------------------------------------------------------------------------------------ far rows
@gpu
def test_rows_behind_the_32_bit_offsets():
    """Logits, gradients and products of more than 2^32 bytes: the last rows are those of a call on them alone, bit for bit."""
    n, v = 70001, 32000
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.empty(n, v, device="cuda", dtype=torch.bfloat16)
    z[:1000].normal_(generator=g)
    for lo in range(1000, n, 1000):
        z[lo:lo + 1000] = z[lo - 1000:lo][: min(1000, n - lo)]
    z[-40:].normal_(generator=g)
    tv, ti = torch.topk(z[:, :64].float(), 5, dim=1)
    last = slice(n - 40, n)
    values, indices = HF.top_logits(z, 7)
    few = HF.top_logits(z[last].clone(), 7)
    assert torch.equal(values[last], few[0]) and torch.equal(indices[last], few[1])
    grads = []
    for rows in (slice(0, n), last):
        leaf = z[rows].detach().requires_grad_()
        HF.distill_loss(leaf, tv[rows], ti[rows], None, 2.0, reduction="sum").backward()
        grads.append(leaf.grad[-40:].clone())
        del leaf
    assert torch.equal(*grads)
    x = rnd((n, 16), 3, torch.bfloat16)
    w, ws = HF.quantize_rows(rnd((v, 16), 4))
    assert torch.equal(HF.linear_int8(x, w, ws)[last], HF.linear_int8(x[last], w, ws))


# ------------------------------------------------------------------------------------------------ together
@gpu
def test_results_do_not_change_from_call_to_call():
    z, tv, ti, y = make_distill(33, 5000, 40, torch.bfloat16, 10)
    w, ws = HF.quantize_rows(rnd((700, 640), 11))
    x = rnd((33, 640), 12)
    first = None
    for _ in range(3):
        leaf = z.detach().requires_grad_()
        loss = HF.distill_loss(leaf, tv, ti, y, 2.0, 0.5, 0.5)
        loss.backward()
        now = [loss.detach(), leaf.grad, *HF.top_logits(z, 40), HF.linear_int8(x, w, ws)]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@gpu
def test_head_selection_and_loss_together_and_captured():
    """A teacher's head in 8 bits, its largest logits, a student's loss and gradient: eager, on another stream, and two captured
    graphs replayed in turn with eager work between (each graph has scratch of its own)."""
    feat = [rnd((40, 640), 20 + i) for i in range(3)]
    student = [rnd((40, 900), 30 + i, torch.bfloat16) for i in range(3)]
    y = torch.randint(0, 900, (40,), generator=torch.Generator().manual_seed(1)).cuda()
    w, ws = HF.quantize_rows(rnd((900, 640), 40, scale=0.1))
    bias = rnd((900,), 41)

    def step(f, z):
        logits = HF.linear_int8(f, w, ws, bias)
        tv, ti = HF.top_logits(logits, 12)
        leaf = z.detach().requires_grad_()
        loss = HF.distill_loss(leaf, tv, ti, y, 2.0, 0.5, 0.5)
        (grad,) = torch.autograd.grad(loss, leaf)
        return logits, tv, ti, loss.detach(), grad

    eager = [[t.clone() for t in step(f, z)] for f, z in zip(feat, student)]
    check_linear(feat[0], w, ws, bias, eager[0][0], torch.float32)
    wv, wi = plain_top(eager[0][0], 12)
    assert torch.equal(eager[0][2].cpu(), wi)
    check_distill(student[0], eager[0][1], eager[0][2], y, 2.0, 0.5, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(feat[1], student[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, eager[1]))

    graphs = []
    for i in range(2):
        f, z = feat[i].clone(), student[i].clone()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            out = step(f, z)
        graphs.append((g, f, z, out))
    for turn in range(3):
        for i, (g, f, z, out) in enumerate(graphs):
            j = (i + turn) % 3
            f.copy_(feat[j])
            z.copy_(student[j])
            g.replay()
            step(feat[2], student[2])                                # eager work between the replays
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager[j])), (turn, i)


@gpu
@pytest.mark.parametrize("int8_head", [False, True])
def test_pretraining_with_a_teacher(int8_head):
    """train(..., teacher=): the step's gradients are the formula's on the teacher's answers, the loop runs, refusals are made."""
    from types import SimpleNamespace

    from subreg_hip import pretrain, synthetic as syn
    from subreg_hip.resnet_language import create_model

    opt = SimpleNamespace(linear_bias=True, hip_dtype="f32", no_dropblock=True, print_freq=100, distill_temperature=2.0)
    torch.manual_seed(0)
    net, old = create_model("resnet12", 20, opt).cuda(), create_model("resnet12", 20, opt).cuda()
    teacher = pretrain.Teacher(old, top=6, int8_head=int8_head)
    x = torch.from_numpy(syn.make_images(3, 4, 32)).cuda()
    y = torch.tensor([0, 5, 7, 19]).cuda()
    values, indices = teacher(x)
    logits = teacher.logits(x)
    wv, wi = plain_top(logits, 6)
    assert torch.equal(indices.cpu(), wi) and torch.equal(values.cpu().double(), wv)
    if int8_head:
        feat = old.hip_backbone().forward(x)
        check_linear(feat, teacher.codes, teacher.scale, old.classifier.bias.detach(), logits, torch.float32)

    out = net.eval()(x).detach().requires_grad_()
    loss = pretrain._distill(teacher, out, x, y, opt)
    loss.backward()
    want, grad = plain_distill(out, values, indices, y, 2.0, 0.5, 0.5)
    row, elem = distill_bounds(out, values, indices, 2.0, 0.5, 0.5)
    close(loss.reshape(1), want.reshape(1), 2 * row)
    close(out.grad, grad, elem)

    net.train()
    before = {n: p.detach().clone() for n, p in net.named_parameters()}
    frozen = {n: p.detach().clone() for n, p in old.state_dict().items()}
    optimizer = pretrain.SGD(net.parameters(), lr=0.01, momentum=0.9, weight_decay=5e-4)
    acc, avg = pretrain.train(1, [(x.cpu(), y.cpu()), (x.cpu(), y.cpu())], net, None, optimizer, opt, log=lambda *a: None, teacher=teacher)
    assert math.isfinite(avg) and 0.0 <= acc <= 100.0
    assert all(not torch.equal(p, before[n]) for n, p in net.named_parameters())
    assert all(torch.equal(p, frozen[n]) for n, p in old.state_dict().items())
    with pytest.raises(ValueError):
        pretrain.train(1, [], net, None, optimizer, SimpleNamespace(hip_graph=True), teacher=teacher)
    with pytest.raises(ValueError):
        pretrain.train(1, [], old, None, optimizer, opt, teacher=teacher)
    with pytest.raises(ValueError):
        pretrain.Teacher(old, top=21)
    with pytest.raises(ValueError):
        pretrain.Teacher(create_model("resnet12", -1, opt))
    small = create_model("resnet12", 10, opt).cuda()
    with pytest.raises(ValueError):
        pretrain.train(1, [], small, None, optimizer, opt, teacher=teacher)


@gpu
def test_documented_lines_run():
    """The lines on the operators in INTEGRATION.md, with an ordinary nn.Linear whose parameters want gradients."""
    import os
    import re

    from conftest import REPO
    with open(os.path.join(REPO, "INTEGRATION.md")) as f:
        (block,) = [b for b in re.findall(r"```python\n(.*?)```", f.read(), re.S) if "HF.quantize_rows" in b]
    names = dict(torch=torch, head=torch.nn.Linear(640, 351).cuda(), features=rnd((16, 640), 1), student_logits=rnd((16, 351), 2).requires_grad_(),
                 target=torch.arange(16).cuda())
    exec(block, names)                                               # (our own text)
    _, want = plain_distill(names["student_logits"], names["values"], names["indices"], names["target"], 2.0, 1.0, 0.5)
    _, elem = distill_bounds(names["student_logits"], names["values"], names["indices"], 2.0, 1.0, 0.5)
    close(names["student_logits"].grad, want, elem)


@gpu
def test_a_teacher_with_two_ranks_uneven_shards():
    """train(..., teacher=, world=2): each rank's gradient carries n_local / n_global, an upstream factor other than 1, so that the sum
    over ranks is the global mean's.  (Both ranks run here one after the other; what they exchange is tests/test_multirank.py's.)"""
    from types import SimpleNamespace

    from subreg_hip import pretrain, synthetic as syn
    from subreg_hip.resnet_language import create_model

    opt = SimpleNamespace(linear_bias=True, hip_dtype="f32", no_dropblock=True, print_freq=100, distill_temperature=2.0)
    torch.manual_seed(0)
    net, old = create_model("resnet12", 20, opt).cuda(), create_model("resnet12", 20, opt).cuda()
    teacher = pretrain.Teacher(old, top=6)
    x, y = torch.from_numpy(syn.make_images(3, 5, 32)), torch.tensor([0, 5, 7, 19, 2])
    outs, grads = [], []
    net.register_forward_hook(lambda m, i, o: outs.append(o.detach()))

    class Watch:
        param_groups = [dict(params=[])]

        def zero_grad(self):
            for p in net.parameters():
                p.grad = None

        def step(self):
            grads.append(net.classifier.bias.grad.clone())

    for rank, cut in ((0, slice(0, 3)), (1, slice(3, 5))):
        pretrain.train(1, [(x, y)], net, None, Watch(), opt, rank=rank, world=2, log=lambda *a: None, teacher=teacher)
        values, indices = teacher(x[cut].cuda())
        out, share = outs[-1], outs[-1].shape[0] / 5
        assert out.shape == (cut.stop - cut.start, 20)
        _, want = plain_distill(out, values, indices, y[cut], 2.0, 0.5, 0.5)
        _, elem = distill_bounds(out, values, indices, 2.0, 0.5, 0.5)
        # three rows at most: their gradients' errors and the additions
        close(grads[-1], share * want.sum(0), share * (3 * elem + 3 * U * want.abs().sum(0)))
