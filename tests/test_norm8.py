"""Group norm with activation, 8-bit checkpoints and the gradients that read them, against plain
evaluations in 64 bits.

Tolerances.  u = 2^-24 is the rounding of fp32 and U that of the element type (bf16 2^-8 / 2, i.e.
finfo.eps / 2).  A result rounded once to its type is off by U |value| (and half the least subnormal);
before that, every fp32 operation adds at most u of its result.  Sums over m values run as a tree of
short sequences: no value passes more than DEPTH roundings, so a sum is off by at most DEPTH u times the
sum of magnitudes.  Where a sum runs sequentially over n rows (weight gradients) the bound is n u times
the sum of magnitudes; exact cases (small integers) carry no tolerance at all."""
import ctypes
import math

import numpy as np
import pytest
import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu"]
U32 = 2.0 ** -24
DEPTH = 96     # 8 rows of a thread, up to 32 batches, 16 row lanes, chunks and channels as a tree
gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def subnormal(dtype):
    f = torch.finfo(dtype)
    return float(f.tiny * f.eps) / 2


# ------------------------------------------------------------------ the checkpoint format in numpy
def quantise_ref(x):
    """(codes (.., C) int, scale bytes, values) of float64 values x (.., C)."""
    x = np.asarray(x, np.float64)
    C = x.shape[-1]
    nb = -(-C // 32)
    codes = np.zeros(x.shape, np.int64)
    scales = np.zeros(x.shape[:-1] + (nb,), np.int64)
    values = np.zeros_like(x)
    for k in range(nb):
        blk = x[..., 32 * k:32 * k + 32]
        ok = np.isfinite(blk).all(-1)
        top = np.abs(np.where(ok[..., None], blk, 0.0)).max(-1)
        m, e = np.frexp(top)
        e = np.where(top == 0, -126, np.maximum(e - 7 + (m > 127 / 128), -126))
        c = np.rint(np.ldexp(np.where(ok[..., None], blk, 0.0), -e[..., None]))
        c = np.where((e == 122)[..., None], np.clip(c, -63, 63), c)
        codes[..., 32 * k:32 * k + 32] = c
        scales[..., k] = np.where(ok, e + 127, 255)
        values[..., 32 * k:32 * k + 32] = np.where(ok[..., None], np.ldexp(c, e[..., None]), np.nan)
    return codes, scales, values


def test_reference_quantiser_bounds():
    """The oracle itself: codes reach at most 127, at least 64 in a block's largest, the error is
    at most half a step and a step at most 2/127 of the block's largest."""
    rng = np.random.default_rng(0)
    x = rng.normal(size=(50, 100)) * np.exp(rng.normal(size=(50, 1)) * 5)
    codes, scales, values = quantise_ref(x)
    assert np.abs(codes).max() <= 127
    for k in range(4):
        blk, c = np.abs(x[:, 32 * k:32 * k + 32]), np.abs(codes[:, 32 * k:32 * k + 32])
        step = np.ldexp(1.0, scales[:, k] - 127)
        assert (c.max(1) >= 63).all()
        assert (np.abs(x[:, 32 * k:32 * k + 32] - values[:, 32 * k:32 * k + 32]).max(1) <= step / 2).all()
        assert (step <= blk.max(1) * 2 / 127 * (1 + 1e-12)).all()


# ------------------------------------------------------------------ refusals
def _lib():
    from graphvae import ops
    return ops._bind()


def _norm_fwd(L, x=16, dtype=0, bs=8, rs=8, B=1, N=1, C=8, G=2, act=1, eps=1e-5, y=16, mean=16, rstd=16, x8=None,
              x8s=None, y8=None, y8s=None, ws=16):
    return L.gvae_group_norm_fwd(x, dtype, bs, rs, None, B, N, C, G, None, None, eps, act, y, mean, rstd, x8, x8s,
                                 y8, y8s, ws, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(y=None), dict(ws=None, N=100000), dict(mean=None), dict(dtype=3),
                                 dict(dtype=-1), dict(B=0), dict(N=0), dict(C=0), dict(G=0), dict(G=3), dict(act=4),
                                 dict(act=-1), dict(rs=-8), dict(bs=-8), dict(eps=0.0), dict(eps=float("nan")),
                                 dict(eps=float("inf")), dict(ws=8), dict(x8=24, x8s=16), dict(y8=8, y8s=16), dict(x8=16), dict(x8s=16), dict(y8=16), dict(y8s=16)])
def test_norm_forward_refusals(bad):
    L = _lib()
    assert _norm_fwd(L, **bad) == -1
    assert b"group_norm_fwd" in L.gvae_last_error()


def test_norm_limits():
    L = _lib()
    assert _norm_fwd(L, B=1 << 20, G=1 << 12, C=1 << 12, rs=1 << 12) == -3
    assert _norm_fwd(L, N=1 << 24, G=1, C=1 << 8, rs=1 << 8) == -3
    assert _norm_fwd(L, B=1 << 22, G=1) == -3 and _norm_fwd(L, C=(1 << 20) + 8, rs=1 << 21, G=1) == -3


@pytest.mark.parametrize("bad", [dict(dy=None), dict(dx=None), dict(x=None), dict(x8=16, x8s=16), dict(x8=16),
                                 dict(x=None, x8=16), dict(x=None, x8s=16), dict(dw=None), dict(db=None),
                                 dict(mean=None), dict(rstd=None), dict(ws=None), dict(dtype=9), dict(G=3), dict(C=0),
                                 dict(rs=-1), dict(drs=-4), dict(bs=-1), dict(dbs=-1), dict(act=7), dict(ws=8),
                                 dict(x=None, x8=8, x8s=16)])
def test_norm_backward_refusals(bad):
    L = _lib()
    k = dict(dy=16, dtype=0, dbs=8, drs=8, x=16, bs=8, rs=8, x8=None, x8s=None, B=1, N=1, C=8, G=2, mean=16, rstd=16,
             act=1, dx=16, dw=16, db=16, ws=16)
    k.update(bad)
    rc = L.gvae_group_norm_bwd(k["dy"], k["dtype"], k["dbs"], k["drs"], k["x"], k["bs"], k["rs"], k["x8"], k["x8s"],
                               None, k["B"], k["N"], k["C"], k["G"], None, None, k["mean"], k["rstd"], k["act"],
                               k["dx"], k["dw"], k["db"], k["ws"], None)
    assert rc == -1 and b"group_norm_bwd" in L.gvae_last_error()


def test_checkpoint_and_wgrad_refusals():
    L = _lib()
    for a in [(None, 0, 1, 8, 8, 16, 16), (16, 3, 1, 8, 8, 16, 16), (16, 0, 0, 8, 8, 16, 16), (16, 0, 1, 0, 8, 16, 16),
              (16, 0, 1, 8, 7, 16, 16), (16, 0, 1, 8, 8, None, 16), (16, 0, 1, 8, 8, 16, None)]:
        assert L.gvae_ckpt8_write(*a, None) == -1, a
        assert b"ckpt8_write" in L.gvae_last_error()
        x, dt, rows, C, ld, codes, scales = a
        assert L.gvae_ckpt8_read(codes, scales, rows, C, x, dt, ld, None) == -1, a
    assert L.gvae_ckpt8_write(16, 0, 1, (1 << 24) + 1, 1 << 25, 16, 16, None) == -3
    for a in [(None, 0, 8, 16, 16, 4, 8, 8, 16, 16, 16), (16, 5, 8, 16, 16, 4, 8, 8, 16, 16, 16),
              (16, 0, 7, 16, 16, 4, 8, 8, 16, 16, 16), (16, 0, 8, None, 16, 4, 8, 8, 16, 16, 16),
              (16, 0, 8, 16, None, 4, 8, 8, 16, 16, 16), (16, 0, 8, 16, 16, 0, 8, 8, 16, 16, 16),
              (16, 0, 8, 16, 16, 4, 0, 8, 16, 16, 16), (16, 0, 8, 16, 16, 4, 8, 0, 16, 16, 16),
              (16, 0, 8, 16, 16, 4, 8, 8, None, 16, 16), (16, 0, 8, 16, 16, 4, 8, 8, 16, 16, None),
              (16, 0, 8, 8, 16, 4, 8, 8, 16, 16, 16), (16, 0, 8, 16, 16, 4, 8, 8, 16, 16, 8)]:
        assert L.gvae_linear_wgrad8(*a, None) == -1, a
        assert b"linear_wgrad8" in L.gvae_last_error()
    for dy_ld, rows, O, I in [(1 << 21, 4, 1 << 21, 8), (1 << 16, 4, 1 << 16, 1 << 16), (1 << 26, 4, 8, 8)]:
        assert L.gvae_linear_wgrad8(16, 0, dy_ld, 16, 16, rows, O, I, 16, 16, 16, None) == -3
    assert L.gvae_ckpt8_write(16, 0, 1 << 40, 1024, 1024, 16, 16, None) == -3
    for n in (L.gvae_group_norm_ws_bytes(1, 0, 0, 1, 1, 1, 0), L.gvae_group_norm_ws_bytes(0, 0, 1, 1, 3, 2, 0), L.gvae_linear_wgrad8_ws_bytes(0, 1, 1)):
        assert n == 0


def test_python_refusals_without_gpu():
    from graphvae import _hip, ops
    x = torch.zeros(2, 4, 32)
    with pytest.raises(_hip.GvaeHipError):
        ops.group_norm_act(x, None, None, 4)
    with pytest.raises(_hip.GvaeHipError):
        ops.checkpoint8(x)
    with pytest.raises(ValueError):
        ops.group_norm_act(x, None, None, 5)
    with pytest.raises(_hip.GvaeHipError):
        ops.group_norm_act(x[0], None, None, 4)
    codes, scales = torch.zeros(2, 4, 32, dtype=torch.int8), torch.zeros(2, 4, 1, dtype=torch.uint8)
    c = ops.Checkpoint8(codes, scales, 20)
    assert c.shape == (2, 4, 20)
    for bad in [(codes, scales, 40), (codes, scales, 16), (codes.float(), scales, 32), (codes, codes, 32),
                (codes, scales, 0), (codes[:, ::2], scales[:, ::2], 32), (codes[:1], scales, 32)]:
        with pytest.raises(_hip.GvaeHipError):
            ops.Checkpoint8(*bad)
    with pytest.raises(_hip.GvaeHipError):
        ops.Checkpoint8(codes, scales, 32, torch.float64)
    with pytest.raises(_hip.GvaeHipError):
        c.read()
    with pytest.raises(_hip.GvaeHipError):
        ops.linear_wgrad8(torch.zeros(2, 4, 8), c)
    with pytest.raises(_hip.GvaeHipError):
        ops.linear_wgrad8(torch.zeros(2, 4, 8), x)


@gpu
def test_python_refusals_on_gpu():
    from graphvae import _hip, ops
    dev = "cuda:0"
    x = torch.zeros(2, 4, 32, device=dev)
    w = torch.ones(32, device=dev)
    E = _hip.GvaeHipError
    for kw in [dict(x=x.double()), dict(x=x.transpose(1, 2)), dict(x=x[:, :, ::2]), dict(x=x[:0]), dict(w=w[:16]),
               dict(w=w.half()), dict(b=w.cpu()), dict(rows=torch.ones(2, device=dev)),
               dict(rows=torch.ones(3, dtype=torch.int32, device=dev))]:
        a = dict(x=x, w=w, b=w, rows=None)
        a.update(kw)
        with pytest.raises(E):
            ops.group_norm_act(a["x"], a["w"], a["b"], 4, rows=a["rows"])
    with pytest.raises(ValueError):
        ops.group_norm_act(x, w, w, 4, act="tanh")
    with pytest.raises(ValueError):
        ops.group_norm_act(x, w, w, 4, eps=0.0)
    r = ops.group_norm_act(x, w, w, 4, keep_x=True)
    dy = torch.zeros_like(x)
    for kw in [dict(dy=dy.half()), dict(dy=dy[:1]), dict(mean=None), dict(rstd=None), dict(x=x.double()), dict(x=x[:, :2]), dict(mean=r.mean[:1]), dict(rstd=r.rstd.double()),
               dict(x=ops.checkpoint8(x[:1])), dict(x=x.cpu())]:
        a = dict(dy=dy, x=x, mean=r.mean, rstd=r.rstd)
        a.update(kw)
        with pytest.raises(E):
            ops.group_norm_act_backward(a["dy"], a["x"], w, w, a["mean"], a["rstd"], 4)
    with pytest.raises(E):
        ops.linear_wgrad8(dy[:1], r.x8)
    with pytest.raises(E):
        ops.linear_wgrad8(dy.transpose(0, 1), r.x8)
    with pytest.raises(E):
        ops.checkpoint8(x.transpose(0, 1))
    with pytest.raises(E):
        ops.checkpoint8(torch.zeros(3, 4, dtype=torch.int32, device=dev))


# ------------------------------------------------------------------ checkpoints
def _special_rows(C, dtype, rng):
    """Rows with every kind of block: ordinary, zeros, subnormal, largest values, ties, not finite."""
    f = torch.finfo(dtype)
    base = rng.normal(size=(12, C))
    x = np.zeros((12, C))
    x[0] = base[0]
    x[2] = base[2] * float(f.tiny) * 0.25
    x[3] = np.where(base[3] > 0, float(f.max), -float(f.max) / 3)
    x[4] = np.rint(base[4] * 40) + 0.5                     # ties
    x[5] = base[5] * 1e4
    x[6] = base[6]
    x[6, rng.integers(C)] = np.inf
    x[7] = base[7]
    x[7, rng.integers(C)] = np.nan
    x[8] = np.where(np.arange(C) % 32 == 0, 127.0, 0.5)    # exactly 127 steps
    x[9] = np.where(np.arange(C) % 32 == 0, 127.5, 1.0)    # just over: the next power
    x[10] = base[10] * np.exp(rng.normal(size=C) * 6)
    x[11] = -np.abs(base[11])
    return torch.from_numpy(x).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 7, 8, 16, 31, 32, 33, 48, 100, 128, 1000, 1024, 2049])
def test_checkpoint_is_the_format(dtype, C):
    from graphvae import ops
    rng = np.random.default_rng(C)
    x = _special_rows(C, dtype, rng)
    codes, scales, values = quantise_ref(x.double().numpy())
    c = ops.checkpoint8(x.cuda())
    ld = -(-C // 16) * 16
    got = c.codes.cpu().numpy().astype(np.int64)
    assert got.shape == (12, ld) and (got[:, C:] == 0).all()
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    assert np.array_equal(got[:, :C], codes)
    for out in DTYPES:
        r = c.read(out).cpu()
        assert r.dtype == out and tuple(r.shape) == (12, C)
        want = torch.from_numpy(values).to(torch.float32)
        if out == torch.float16:
            want = torch.where(want.isnan(), want, want.clamp(-65504.0, 65504.0))
        assert torch.equal(torch.nan_to_num(r.float(), nan=7e37), torch.nan_to_num(want.to(out).float(), nan=7e37))
    assert c.read().dtype == dtype


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_strides_and_sizes(dtype):
    from graphvae import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    for rows, C, ld, off in [(1, 1, 1, 0), (1, 64, 64, 0), (5, 40, 64, 0), (3, 33, 35, 1), (1000, 37, 41, 3),
                             (4097, 128, 128, 0), (2, 70000, 70000, 0)]:
        buf = torch.randn(rows * ld + off, generator=g, device="cuda").to(dtype)
        x = buf[off:].view(rows, ld)[:, :C]
        c = ops.checkpoint8(x)
        _, scales, values = quantise_ref(x.double().cpu().numpy())
        assert np.array_equal(c.scales.cpu().numpy(), scales)
        assert np.array_equal(c.read(torch.float32).double().cpu().numpy(), values)
    x = torch.randn(2, 3, 4, 40, generator=g, device="cuda").to(dtype)
    assert ops.checkpoint8(x).shape == (2, 3, 4, 40)
    v = torch.randn(45, generator=g, device="cuda").to(dtype)
    assert torch.equal(ops.checkpoint8(v).read(), ops.checkpoint8(v.view(1, 45)).read()[0])


@gpu
def test_checkpoint_past_32_bit_offsets():
    """More than 2^32 elements: the last rows are read and written where they belong."""
    from graphvae import ops
    rows, C = (1 << 22) + 37, 1024
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    x[-40:] = torch.randn(40, C, device="cuda").to(torch.bfloat16)
    x[:5] = torch.randn(5, C, device="cuda").to(torch.bfloat16)
    c = ops.checkpoint8(x)
    r = c.read()
    assert torch.equal(r[-40:], ops.checkpoint8(x[-40:]).read())
    assert torch.equal(r[:5], ops.checkpoint8(x[:5]).read())
    assert not r[5:-40].any()


# ------------------------------------------------------------------ group norm
def act_ref(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    return z


def slope_ref(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z) if act == "none" else (z > 0).to(z.dtype)


def per_channel(t, C):
    return t.repeat_interleave(C // t.shape[1], 1)[:, None, :]


def norm_ref(x, w, b, G, act, eps, rows):
    """y, mean, rstd and the bound on y's fp32 error, in float64 on the CPU."""
    B, N, C = x.shape
    x, w, b = x.double(), w.double(), b.double()
    live = (torch.arange(N)[None, :, None] < rows[:, None, None])
    n = rows.clamp(min=1).double()[:, None] * (C // G)
    xs = torch.where(live, x, torch.zeros_like(x))
    mean = xs.view(B, N, G, -1).sum((1, 3)) / n
    d = torch.where(live, x - per_channel(mean, C), torch.zeros_like(x))
    var = d.square().view(B, N, G, -1).sum((1, 3)) / n
    rstd = (var + eps).rsqrt()
    h = d * per_channel(rstd, C)
    z = h * w + b
    y = torch.where(live, act_ref(z, act), torch.zeros_like(z))
    # mean off by DEPTH u of the mean magnitude; the centred square sum by DEPTH u of itself plus the
    # square of the mean's error, so rstd by half that relatively; four more roundings to z, and the
    # activation a few of its own (slope at most 1.13)
    dmean = (DEPTH + 2) * U32 * xs.abs().view(B, N, G, -1).sum((1, 3)) / n
    drel = (DEPTH / 2 + 4) * U32 + (dmean * rstd) ** 2
    dh = per_channel(dmean * rstd, C) + h.abs() * per_channel(drel, C) + 2 * U32 * (x.abs() * per_channel(rstd, C) + h.abs())
    tol = 1.13 * (dh * w.abs() + 3 * U32 * (z.abs() + b.abs() + (h * w).abs())) + 12 * U32 * (z.abs() + 1e-30)
    return y, mean, rstd, torch.where(live, tol, torch.zeros_like(tol)), dmean, drel


def make_x(B, N, C, dtype, seed, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, N, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + mean * torch.randn(C, generator=g) + 0.25
    w = 1 + 0.3 * torch.randn(C, generator=g)
    b = 0.3 * torch.randn(C, generator=g)
    rows = torch.randint(0, N + 1, (B,), generator=g, dtype=torch.int32)
    rows[0] = 0
    rows[-1] = N
    if B > 2:
        rows[1] = 1
    dy = torch.randn(B, N, C, generator=g)
    return x.to(dtype), w, b, rows, dy.to(dtype)


# (graphs, rows, channels, groups): one row, one channel, groups that split a vector or span many,
# rows that do not fill a work-group, long row axes, wide rows, a batch of many small graphs
SHAPES = [(1, 1, 1, 1), (2, 1, 32, 1), (3, 1, 700, 7), (3, 20, 128, 8), (4, 5, 6, 3), (5, 33, 45, 9), (2, 126, 128, 128),
          (3, 17, 96, 1), (2, 1000, 40, 8), (2, 777, 33, 11), (1, 5000, 64, 2), (2, 65, 1536, 32), (1, 3, 4100, 5),
          (1, 2, 9000, 1), (300, 7, 24, 3), (2, 300, 520, 4), (1, 20000, 8, 1), (3, 40, 2500, 2500)]


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_forward(shape, dtype):
    from graphvae import ops
    B, N, C, G = shape
    for k, act in enumerate(ACTS):
        x, w, b, rows, _ = make_x(B, N, C, dtype, 100 * k + C)
        if k % 2 and B > 0:
            live = rows
        else:
            live = torch.full((B,), N, dtype=torch.int32)
        xin = x.clone()
        dead = torch.arange(N)[None, :, None] >= live[:, None, None]
        xin = torch.where(dead, torch.full_like(xin, float("nan")), xin)   # never read
        r = ops.group_norm_act(xin.cuda(), w.cuda(), b.cuda(), G, act=act, rows=live.cuda() if k % 2 else None,
                               keep_x=k > 1, keep_y=k != 0)
        y, mean, rstd, tol, dmean, drel = norm_ref(torch.where(dead, torch.zeros_like(x), x), w, b, G, act, 1e-5, live)
        assert r.y.dtype == dtype and tuple(r.y.shape) == (B, N, C)
        err = (r.y.cpu().double() - y).abs()
        bound = half_step(dtype) * y.abs() + (1 + half_step(dtype)) * tol + subnormal(dtype)
        assert (err <= bound).all(), (act, float((err - bound).max()))
        assert not r.y.cpu()[dead.expand_as(y)].any()
        assert ((r.mean.cpu().double() - mean).abs() <= dmean + 2 * U32 * mean.abs()).all()
        assert ((r.rstd.cpu().double() / rstd - 1).abs() <= drel + 4 * U32).all()
        # checkpoints: what checkpoint8 makes of the same tensors, bit for bit
        if k > 1:
            c = ops.checkpoint8(torch.where(dead, torch.zeros_like(x), x).cuda())
            assert torch.equal(c.codes, r.x8.codes) and torch.equal(c.scales, r.x8.scales)
            assert r.x8.dtype == dtype
        if k != 0:
            c = ops.checkpoint8(r.y)
            assert torch.equal(c.codes, r.y8.codes) and torch.equal(c.scales, r.y8.scales)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_large_mean(dtype):
    """Values far from zero (mean of 300 and more standard deviations): no uncentred square is summed.  x8
    of a constant block, and a group of equal values (variance 0) stay finite."""
    from graphvae import ops
    for N, C, G in [(64, 64, 4), (3000, 32, 2)]:
        x, w, b, _, _ = make_x(2, N, C, dtype, 5, mean=0.0)
        x = (x.float() + 400.0).to(dtype)
        x[0, :, :C // G] = 3.0
        rows = torch.full((2,), N, dtype=torch.int32)
        r = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act="none")
        y, mean, rstd, tol, dmean, drel = norm_ref(x, w, b, G, "none", 1e-5, rows)
        err = (r.y.cpu().double() - y).abs()
        assert (err <= half_step(dtype) * y.abs() + 1.01 * tol + subnormal(dtype)).all()
        assert ((r.rstd.cpu().double() / rstd - 1).abs() <= drel + 4 * U32).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_not_finite(dtype):
    """An infinity or a NaN spoils its own group of its own graph only, in every row of it."""
    from graphvae import ops
    for N, C, G in [(10, 24, 3), (2000, 24, 3)]:
        x, w, b, _, _ = make_x(3, N, C, dtype, 8)
        clean = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act="relu", keep_x=True, keep_y=True)
        for bad in (float("nan"), float("inf"), float("-inf")):
            xb = x.clone()
            xb[1, N // 2, C // G + 1] = bad
            r = ops.group_norm_act(xb.cuda(), w.cuda(), b.cuda(), G, act="relu", keep_x=True, keep_y=True)
            spoiled = torch.zeros(3, N, C, dtype=torch.bool)
            spoiled[1, :, C // G:2 * C // G] = True
            assert r.y.cpu()[spoiled].isnan().all()
            assert torch.equal(r.y.cpu()[~spoiled], clean.y.cpu()[~spoiled])
            assert r.x8.read().cpu()[1, N // 2].isnan().all() and not r.x8.read().cpu()[0].isnan().any()
            assert r.y8.read().cpu()[1].isnan().all() and not r.y8.read().cpu()[2].isnan().any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_strides(dtype):
    """Any batch and row stride, odd alignments, a batch that is one graph expanded."""
    from graphvae import ops
    B, N, C, G = 3, 37, 40, 5
    g = torch.Generator(device="cuda").manual_seed(3)
    w, b = torch.randn(C, generator=g, device="cuda"), torch.randn(C, generator=g, device="cuda")
    buf = torch.randn(B, N + 3, C + 5, generator=g, device="cuda").to(dtype)
    views = [buf[:, 1:N + 1, 3:3 + C], buf[:, :N, :C], buf.transpose(0, 1)[:B, :B, 1:C + 1],
             buf[:1, :N, :C].expand(4, N, C), buf[:, :1, 1:1 + C], buf[1:2, 2:3, :C], buf[:, :1, :C].expand(B, N, C),
             buf[:1, :1, 5:5 + C].expand(B, 700, C)]
    for x in views:
        dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        r, c = (ops.group_norm_act(t, w, b, G, act="silu", keep_x=True) for t in (x, x.contiguous()))
        assert torch.equal(r.y, c.y) and torch.equal(r.x8.codes, c.x8.codes)
        one = dy[:, :1, :].expand(x.shape) if x.shape[1] == 1 else dy[:1].expand(x.shape)
        rows_one = dy[:, :1, :].expand(x.shape)
        for gy in (dy, one, rows_one):
            a = ops.group_norm_act_backward(gy, x, w, b, r.mean, r.rstd, G, act="silu")
            e = ops.group_norm_act_backward(gy.contiguous(), x.contiguous(), w, b, r.mean, r.rstd, G, act="silu")
            assert all(torch.equal(p, q) for p, q in zip(a, e))


def bwd_ref(dy, x, w, b, mean, rstd, G, act, rows):
    """dx, dw, db and their bounds in float64; x: the values the backward works on.  A ReLU's branch is
    that of the fp32 z = ((x - mean) * rstd) * w + b, every operation rounded."""
    B, N, C = dy.shape
    live = (torch.arange(N)[None, :, None] < rows[:, None, None])
    zero = torch.zeros(B, N, C, dtype=torch.float64)
    m32, r32 = per_channel(mean, C), per_channel(rstd, C)
    z32 = ((x.float() - m32) * r32) * w + b
    x, dy, w, b = x.double(), dy.double(), w.double(), b.double()
    m, r = m32.double(), r32.double()
    h = (x - m) * r
    z = h * w + b
    s = slope_ref(z32.double() if act == "relu" else z, act)
    dz = torch.where(live, dy * s, zero)
    h = torch.where(live, h, zero)
    n = rows.clamp(min=1).double()[:, None] * (C // G)

    def group(t):
        return per_channel(t.view(B, N, G, -1).sum((1, 3)) / n, C)

    a1, a2 = group(dz * w), group(dz * w * h)
    dx = torch.where(live, r * (dz * w - a1 - h * a2), zero)
    # z off by a few roundings of its terms; a smooth activation's slope by 1.2 times that (its
    # second derivative) and a few roundings of its own
    smooth = act in ("silu", "gelu")
    ez = 4 * U32 * ((x.abs() + m.abs()) * r * w.abs() + (h * w).abs() + b.abs()) if smooth else zero
    edz = torch.where(live, dy.abs() * ((1.2 * ez + 16 * U32) if smooth else zero + U32), zero)
    eh = torch.where(live, 3 * U32 * (x.abs() + m.abs()) * r, zero)
    t1 = edz + DEPTH * U32 * dz.abs()
    t2 = edz * h.abs() + dz.abs() * eh + DEPTH * U32 * (dz * h).abs()
    wa = w.abs()
    e1, e2 = group(t1 * wa), group(t2 * wa)
    edx = torch.where(live, r * (edz * wa + e1 + h.abs() * e2 + eh * a2.abs()
                                 + 4 * U32 * ((dz * w).abs() + a1.abs() + (h * a2).abs())), zero)
    return dx, (dz * h).sum((0, 1)), dz.sum((0, 1)), edx, t2.sum((0, 1)), t1.sum((0, 1))


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_backward(shape, dtype):
    from graphvae import ops
    B, N, C, G = shape
    for k, act in enumerate(ACTS):
        for kept in (False, True):
            x, w, b, rows, dy = make_x(B, N, C, dtype, 100 * k + C + 1)
            if not (k % 2) ^ kept:
                rows = torch.full((B,), N, dtype=torch.int32)
            dead = torch.arange(N)[None, :, None] >= rows[:, None, None]
            x = torch.where(dead, torch.zeros_like(x), x)
            _, mean, rstd, _, _, _ = norm_ref(x, w, b, G, act, 1e-5, rows)
            mean, rstd = mean.float(), rstd.float()
            nan = torch.full_like(x, float("nan"))
            arg = ops.checkpoint8(x.cuda()) if kept else torch.where(dead, nan, x).cuda()
            used = arg.read(torch.float32).cpu() if kept else x
            got = ops.group_norm_act_backward(torch.where(dead, nan, dy).cuda(), arg, w.cuda(), b.cuda(), mean.cuda(),
                                              rstd.cuda(), G, act=act, rows=rows.cuda())
            dx, dw, db, edx, edw, edb = bwd_ref(dy, used, w, b, mean, rstd, G, act, rows)
            assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == torch.float32
            err = (got[0].cpu().double() - dx).abs()
            bound = half_step(dtype) * dx.abs() + (1 + half_step(dtype)) * edx + subnormal(dtype)
            assert (err <= bound).all(), (act, kept, float((err - bound).max()))
            assert not got[0].cpu()[dead.expand_as(x)].any()
            # (the sum over graphs adds at most 64 + 16 roundings in sequence)
            assert ((got[1].cpu().double() - dw).abs() <= edw * (1 + 80 / DEPTH) + 1e-30).all()
            assert ((got[2].cpu().double() - db).abs() <= edb * (1 + 80 / DEPTH) + 1e-30).all()


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_group_norm_backward_against_differences(act):
    """Directional derivatives of the forward kernel along random directions, against the backward's
    inner products.  The reference's own difference quotient in float64 says what the step leaves out."""
    from graphvae import ops
    B, N, C, G = 3, 21, 24, 3
    x, w, b, rows, dy = make_x(B, N, C, torch.float32, 11)
    g = torch.Generator().manual_seed(12)
    live = torch.arange(N)[None, :, None] < rows[:, None, None]
    x = torch.where(live, x, torch.zeros_like(x))
    dy = torch.where(live, dy, torch.zeros_like(dy))
    r = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act=act, rows=rows.cuda())
    dx, dw, db = (t.cpu().double() for t in ops.group_norm_act_backward(
        dy.cuda(), x.cuda(), w.cuda(), b.cuda(), r.mean, r.rstd, G, act=act, rows=rows.cuda()))
    step = 2.0 ** -7
    for which in range(3):
        d = [torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)]
        d[which] = torch.randn(d[which].shape, generator=g)
        ends, refs, tols = [], [], []
        for s in (1, -1):
            args = [t + s * step * e for t, e in zip((x, w, b), d)]
            y = ops.group_norm_act(*(t.cuda() for t in args), G, act=act, rows=rows.cuda()).y
            yr, _, _, tol, _, _ = norm_ref(*args, G, act, 1e-5, rows)
            ends.append(float((y.cpu().double() * dy.double()).sum()))
            refs.append(float((yr * dy.double()).sum()))
            tols.append(float(((tol + U32 * yr.abs()) * dy.double().abs()).sum()))
        quotient, ref = ((e[0] - e[1]) / (2 * step) for e in (ends, refs))
        inner = sum(float((t * e.double()).sum()) for t, e in zip((dx, dw, db), d))
        xr = [t.double().requires_grad_() for t in (x, w, b)]
        yr, *_ = norm_ref(*xr, G, act, 1e-5, rows)
        exact = sum(float((t * e.double()).sum()) for t, e in
                    zip(torch.autograd.grad((yr * dy.double()).sum(), xr), d))
        noise = sum(tols) / (2 * step)
        assert abs(quotient - ref) <= noise
        # (what the kernels' gradient and the formula's differ by: the backward's bound along d)
        _, _, _, edx, edw, edb = bwd_ref(dy, x, w, b, r.mean.cpu(), r.rstd.cpu(), G, act, rows)
        bound = sum(float(((e * 2 + U32 * t.abs()) * k.double().abs()).sum()) for e, t, k in
                    zip((edx, edw, edb), (dx, dw, db), d))
        # mean and rstd enter the backward as fp32: each shifts h by a rounding of the sums behind it
        shift = DEPTH * U32 * 4 * float((dy.abs() * per_channel(r.rstd.cpu(), C) * (1 + x.abs())).sum()) \
            * float(max(k.abs().max() for k in d))
        assert abs(inner - exact) <= bound + shift
        assert abs(quotient - inner) <= noise + abs(ref - exact) + bound + shift


# ------------------------------------------------------------------ weight gradients
WG_SHAPES = [(1, 1, 1), (1, 40, 33), (2, 128, 128), (15, 17, 16), (16, 16, 48), (63, 65, 31), (64, 128, 64),
             (65, 129, 130), (500, 100, 36), (1000, 3, 257), (2049, 70, 5), (333, 515, 387), (129, 1, 300)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wgrad_integers_are_exact(dtype):
    """Small integers: every product and every sum is exact in fp32, so the result is exact, and exact
    again in the element type where it fits its significand (asserted through fp32 rounding)."""
    from graphvae import ops
    rng = np.random.default_rng(2)
    for M, O, I in WG_SHAPES:
        dy = rng.integers(-8, 9, (M, O)).astype(np.float64)
        codes, scales, x = quantise_ref(rng.integers(-127, 128, (M, I)).astype(np.float64))
        c = ops.checkpoint8(torch.from_numpy(x).float().cuda())
        dw, db = ops.linear_wgrad8(torch.from_numpy(dy).to(dtype).cuda(), c)
        want, wb = torch.from_numpy(dy.T @ x), torch.from_numpy(dy.sum(0))
        assert float(want.abs().max()) < 2 ** 24
        assert dw.dtype == dtype and torch.equal(dw.cpu(), want.float().to(dtype)), (M, O, I)
        assert torch.equal(db.cpu(), wb.float().to(dtype)), (M, O, I)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", WG_SHAPES)
def test_wgrad_against_64_bits(dtype, shape):
    from graphvae import ops
    M, O, I = shape
    g = torch.Generator().manual_seed(M + O + I)
    dy = (torch.randn(M, O, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    x = torch.randn(M, I, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    c = ops.checkpoint8(x.to(dtype).cuda())
    xd = c.read(torch.float32).cpu().double()
    dw, db = ops.linear_wgrad8(dy.cuda(), c)
    want, mag = dy.double().t() @ xd, dy.double().abs().t() @ xd.abs()
    n = M + 8      # roundings a sum over M exact products can pass through
    assert ((dw.cpu().double() - want).abs() <= half_step(dtype) * want.abs() + 1.01 * n * U32 * mag
            + subnormal(dtype)).all()
    sb = dy.double().sum(0)
    assert ((db.cpu().double() - sb).abs() <= half_step(dtype) * sb.abs() + 1.01 * n * U32 * dy.double().abs().sum(0)
            + subnormal(dtype)).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wgrad_single_row_products(dtype):
    """One row: an element is one product (and zeros), so it carries one product's rounding: the gradient
    enters with all its bits whatever its type.  Three pieces of an fp32 gradient are added: 3 u."""
    from graphvae import ops
    g = torch.Generator().manual_seed(9)
    dy = (torch.randn(1, 130, generator=g) * torch.exp(5 * torch.randn(1, 130, generator=g))).to(dtype)
    c = ops.checkpoint8((torch.randn(1, 70, generator=g)).cuda())
    xd = c.read(torch.float32).cpu().double()
    dw, _ = ops.linear_wgrad8(dy.cuda(), c)
    want = dy.double().t() @ xd
    near = (dw.cpu().double() - want).abs() <= (half_step(dtype) + 3 * U32) * want.abs() + subnormal(dtype)
    # (half ends at 65504: 65520 or more is an infinity in it, at no finite distance from its value, and two
    # of these gradients are infinite as halves: infinity times a code, NaN where the code is 0)
    beyond = ~(want.abs() < 65520.0) & (dtype == torch.float16)
    assert near[~beyond].all()
    torch.testing.assert_close(dw.cpu()[beyond], want.to(dtype)[beyond], rtol=0, atol=0, equal_nan=True)


@gpu
def test_wgrad_strides_lead_axes_and_not_finite():
    from graphvae import ops
    g = torch.Generator(device="cuda").manual_seed(4)
    for dtype in DTYPES:
        buf = torch.randn(6 * 50, 77, generator=g, device="cuda").to(dtype)
        c3 = ops.checkpoint8(torch.randn(6, 50, 64, generator=g, device="cuda").to(dtype))
        c2 = ops.Checkpoint8(c3.codes.view(300, 64), c3.scales.view(300, 2), 64)
        for o, off in ((77, 0), (40, 1), (33, 40)):
            dy = buf[:, off:off + o]
            a, e = ops.linear_wgrad8(dy, c2), ops.linear_wgrad8(dy.contiguous(), c2)
            assert all(torch.equal(p, q) for p, q in zip(a, e))
            d3 = ops.linear_wgrad8(dy.contiguous().view(6, 50, o), c3)
            assert all(torch.equal(p, q) for p, q in zip(a, d3))
        # a block that is not finite reaches the 32 columns it belongs to, an infinite gradient its row
        x = torch.randn(300, 64, generator=g, device="cuda").to(dtype)
        x[123, 40] = float("inf")
        dy = buf[:, :20].clone()
        dw, db = ops.linear_wgrad8(dy, ops.checkpoint8(x))
        assert dw[:, 32:].isnan().all() and not dw[:, :32].isnan().any() and not db.isnan().any()
        dy[7, 3] = float("nan")
        dw, db = ops.linear_wgrad8(dy, ops.checkpoint8(x))
        assert dw[3].isnan().all() and not dw[4, :32].isnan().any() and db[3].isnan() and not db[4].isnan()


# ------------------------------------------------------------------ together
def _layer(ops, x, W, w, b, G, rows, dy):
    """One linear + norm + ReLU layer trained from its checkpoints, as a user runs it: returns every
    result."""
    B, N, I = x.shape
    x8 = ops.checkpoint8(x)
    h = (x.view(-1, I).float() @ W.t().float()).to(x.dtype).view(B, N, -1)
    r = ops.group_norm_act(h, w, b, G, rows=rows, keep_x=True, keep_y=True)
    dh, dw, db = ops.group_norm_act_backward(dy, r.x8, w, b, r.mean, r.rstd, G, rows=rows)
    gW, gB = ops.linear_wgrad8(dh, x8)
    return [r.y, r.mean, r.rstd, r.y8.read(), dh, dw, db, gW, gB]


def _layer_inputs(dtype, seed, B=5, N=60, I=48, O=96):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, N, I, generator=g, device="cuda").to(dtype)
    W = torch.randn(O, I, generator=g, device="cuda").to(dtype) * 0.2
    w, b = 1 + 0.1 * torch.randn(O, generator=g, device="cuda"), 0.1 * torch.randn(O, generator=g, device="cuda")
    rows = torch.randint(0, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    dy = torch.randn(B, N, O, generator=g, device="cuda").to(dtype)
    return x, W, w, b, 6, rows, dy


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_from_checkpoints(dtype):
    """A run of the operators together against the same formulas in 64 bits on the checkpointed values."""
    from graphvae import ops
    x, W, w, b, G, rows, dy = _layer_inputs(dtype, 1)
    y, mean, rstd, y8, dh, dw, db, gW, gB = (t.cpu() for t in _layer(ops, x, W, w, b, G, rows, dy))
    h = (x.view(-1, 48).float() @ W.t().float()).to(dtype).view(5, 60, 96).cpu()
    rows = rows.cpu()
    live = torch.arange(60)[None, :, None] < rows[:, None, None]
    h = torch.where(live, h, torch.zeros_like(h))
    yr, mr, rr, tol, _, _ = norm_ref(h, w.cpu(), b.cpu(), G, "relu", 1e-5, rows)
    assert ((y.double() - yr).abs() <= half_step(dtype) * yr.abs() + 1.01 * tol + subnormal(dtype)).all()
    h8 = torch.from_numpy(quantise_ref(h.double().numpy())[2]).float()
    dxr, dwr, dbr, edx, edw, edb = bwd_ref(dy.cpu(), h8, w.cpu(), b.cpu(), mean, rstd, G, "relu", rows)
    assert ((dh.double() - dxr).abs() <= half_step(dtype) * dxr.abs() + 1.01 * edx + subnormal(dtype)).all()
    assert ((dw.double() - dwr).abs() <= 2 * edw).all() and ((db.double() - dbr).abs() <= 2 * edb).all()
    x8 = torch.from_numpy(quantise_ref(x.double().cpu().numpy())[2]).view(300, 48)
    d2 = dh.double().view(300, 96)
    want, mag = d2.t() @ x8, d2.abs().t() @ x8.abs()
    assert ((gW.double() - want).abs() <= half_step(dtype) * want.abs() + 310 * U32 * mag + subnormal(dtype)).all()
    assert torch.equal(y8.float(), torch.from_numpy(quantise_ref(y.double().numpy())[2]).to(dtype).float())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dtype):
    """The whole layer recorded into a graph: every replay on new inputs equals the eager result, with
    eager work on the same operators between the replays; the same on a stream of its own."""
    from graphvae import ops
    static = _layer_inputs(dtype, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _layer(ops, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(ops, *static)
    for seed in (3, 4, 5, 6):
        fresh = _layer_inputs(dtype, seed)
        want = _layer(ops, *fresh)
        for s, f in zip(static, fresh):
            if isinstance(s, torch.Tensor):
                s.copy_(f)
        torch.cuda.synchronize()
        graph.replay()
        other = _layer(ops, *_layer_inputs(dtype, seed + 100))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), seed
        assert not torch.equal(other[0], want[0])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = _layer(ops, *fresh)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(again, want)), seed


@gpu
def test_results_repeat_bit_for_bit():
    from graphvae import ops
    for dtype in DTYPES:
        args = _layer_inputs(dtype, 7, B=40, N=150, I=64, O=192)
        first = _layer(ops, *args)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, _layer(ops, *args)))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1024, 256, 256), (1500, 300, 260), (3001, 515, 387), (70000, 40, 30),
                                   (20000, 128, 128), (4100, 257, 1000), (100001, 260, 511), (66701, 500, 760),
                                   (200000, 256, 256)])
def test_wgrad_large_tiles_and_many_parts(dtype, shape):
    """Sizes that take the larger tiles, several of them, and many row ranges: against 64 bits, and
    small integers exactly."""
    from graphvae import ops
    M, O, I = shape
    g = torch.Generator(device="cuda").manual_seed(M + O)
    codes = torch.randint(-127, 128, (M, -(-I // 16) * 16), generator=g, device="cuda", dtype=torch.int8)
    codes[:, I:] = 0
    c = ops.Checkpoint8(codes, torch.full((M, -(-I // 32)), 127, dtype=torch.uint8, device="cuda"), I)
    x = codes[:, :I].double()
    dy = torch.randint(-1, 2, (M, O), generator=g, device="cuda").to(dtype)
    dw, db = ops.linear_wgrad8(dy, c)
    want = dy.double().t() @ x
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(dw, want.float().to(dtype)) and torch.equal(db, dy.double().sum(0).float().to(dtype))
    scales = torch.randint(120, 130, (M, -(-I // 32)), generator=g, device="cuda", dtype=torch.uint8)
    c = ops.Checkpoint8(codes, scales, I)
    x = x * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, :I]
    dy = torch.randn(M, O, generator=g, device="cuda").to(dtype)
    dw, db = ops.linear_wgrad8(dy, c)
    want, mag = dy.double().t() @ x, dy.double().abs().t() @ x.abs()
    bound = 1.01 * (M + 8) * U32 * mag
    near = (dw.double() - want).abs() <= half_step(dtype) * want.abs() + bound + subnormal(dtype)
    # (half ends at 65504, and 65520 or more is an infinity in it, at no finite distance: of the sums over
    # 70000 rows some are; within `bound` of that border either answer is right)
    beyond = (want.abs() + bound >= 65520.0) & (dtype == torch.float16)
    assert near[~beyond].all()
    sure = beyond & (want.abs() - bound >= 65520.0)
    assert torch.equal(dw[sure], want.to(dtype)[sure]) and (dw[beyond].abs() >= 65504.0 - 2 * bound[beyond]).all()
    sb = dy.double().sum(0)
    assert ((db.double() - sb).abs() <= half_step(dtype) * sb.abs() + 1.01 * (M + 8) * U32 * dy.double().abs().sum(0)
            + subnormal(dtype)).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(200, 400, 64, 4), (40, 1000, 96, 6), (2, 70000, 32, 4), (1200, 9, 40, 8),
                                   (1100, 3, 5, 5), (9, 4000, 45, 9), (130, 600, 33, 1), (4, 1200, 16, 2),
                                   (40, 300, 512, 16), (130, 200, 60, 6)])
def test_group_norm_forms(dtype, shape):
    """Sizes around the resident and the split form's borders, forward and backward, from the tensor and
    from its checkpoint."""
    from graphvae import ops
    B, N, C, G = shape
    x, w, b, rows, dy = make_x(B, N, C, dtype, C)
    live = torch.arange(N)[None, :, None] < rows[:, None, None]
    x = torch.where(live, x, torch.zeros_like(x))
    r = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act="silu", rows=rows.cuda(), keep_x=True, keep_y=True)
    y, mean, rstd, tol, dmean, drel = norm_ref(x, w, b, G, "silu", 1e-5, rows)
    assert ((r.y.cpu().double() - y).abs() <= half_step(dtype) * y.abs() + 1.01 * tol + subnormal(dtype)).all()
    assert ((r.mean.cpu().double() - mean).abs() <= dmean + 2 * U32 * mean.abs()).all()
    assert ((r.rstd.cpu().double() / rstd - 1).abs() <= drel + 4 * U32).all()
    for got, src in ((r.x8, x.cuda()), (r.y8, r.y)):
        c = ops.checkpoint8(src)
        assert torch.equal(c.codes, got.codes) and torch.equal(c.scales, got.scales)
    for arg, used in ((x.cuda(), x), (r.x8, r.x8.read(torch.float32).cpu())):
        got = ops.group_norm_act_backward(dy.cuda(), arg, w.cuda(), b.cuda(), r.mean, r.rstd, G, act="silu",
                                          rows=rows.cuda())
        dx, dw, db, edx, edw, edb = bwd_ref(dy, used, w, b, r.mean.cpu(), r.rstd.cpu(), G, "silu", rows)
        assert ((got[0].cpu().double() - dx).abs() <= half_step(dtype) * dx.abs() + 1.01 * edx + subnormal(dtype)).all()
        assert ((got[1].cpu().double() - dw).abs() <= 2 * edw).all() and ((got[2].cpu().double() - db).abs() <= 2 * edb).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_empty_batches_and_row_counts_out_of_range(dtype):
    """No live row anywhere: zeros everywhere, gradients 0.  Row counts under 0 and over N count as 0 and N."""
    from graphvae import ops
    for B, N, C, G in [(2, 7, 24, 3), (2, 9000, 24, 3), (1, 50, 16, 2)]:
        x, w, b, _, dy = make_x(B, N, C, dtype, 4)
        x, w, b, dy = x.cuda(), w.cuda(), b.cuda(), dy.cuda()
        none = torch.zeros(B, dtype=torch.int32, device="cuda")
        r = ops.group_norm_act(x, w, b, G, act="gelu", rows=none, keep_x=True, keep_y=True)
        assert not r.y.any() and not r.x8.read().any() and not r.y8.read().any() and not r.mean.any()
        assert (r.rstd.double() - 1e-5 ** -0.5).abs().max() <= 4 * U32 * 1e-5 ** -0.5
        for arg in (x, r.x8):
            got = ops.group_norm_act_backward(dy, arg, w, b, r.mean, r.rstd, G, act="gelu", rows=none)
            assert not any(t.any() for t in got)
        odd = torch.tensor([-5, N + 100][:B], dtype=torch.int32, device="cuda")
        fit = torch.tensor([0, N][:B], dtype=torch.int32, device="cuda")
        a, e = (ops.group_norm_act(x, w, b, G, rows=k) for k in (odd, fit))
        assert torch.equal(a.y, e.y) and torch.equal(a.rstd, e.rstd)
        a, e = (ops.group_norm_act_backward(dy, x, w, b, a.mean, a.rstd, G, rows=k) for k in (odd, fit))
        assert all(torch.equal(p, q) for p, q in zip(a, e))


@gpu
def test_group_norm_without_parameters():
    from graphvae import ops
    for shape in [(3, 40, 48, 6), (2, 9000, 20, 4)]:
        x, _, _, rows, dy = make_x(*shape[:3], torch.float32, 6)
        C, G = shape[2:]
        one, zero = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
        a, e = (ops.group_norm_act(x.cuda(), w, b, G, act="silu", rows=rows.cuda()) for w, b in ((None, None), (one, zero)))
        assert torch.equal(a.y, e.y)
        a, e = (ops.group_norm_act_backward(dy.cuda(), x.cuda(), w, b, a.mean, a.rstd, G, act="silu", rows=rows.cuda())
                for w, b in ((None, None), (one, zero)))
        assert all(torch.equal(p, q) for p, q in zip(a, e))


@gpu
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -60, 2.0 ** 100])
def test_wgrad_far_exponents(scale):
    """Gradients far from one keep all their bits: the pieces of an fp32 gradient reach 2^-16 below it, which
    for 2^-100 is still a normal number."""
    from graphvae import ops
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(1, 64, generator=g) * scale
    c = ops.checkpoint8(torch.randn(1, 40, generator=g).cuda())
    dw, db = ops.linear_wgrad8(dy.cuda(), c)
    want = dy.double().t() @ c.read(torch.float32).cpu().double()
    assert ((dw.cpu().double() - want).abs() <= 4 * U32 * want.abs()).all() and torch.equal(db.cpu(), dy[0])


@gpu
def test_checkpoint_copies_and_views():
    import copy
    from graphvae import ops
    x = torch.randn(4, 5, 70, device="cuda")
    c = ops.checkpoint8(x)
    d = copy.deepcopy(c)
    want = c.read()
    c.codes.zero_()
    assert torch.equal(d.read(), want) and not c.read().any() and d.shape == x.shape and d.dtype == x.dtype
    e = ops.Checkpoint8(d.codes[1:3], d.scales[1:3], 70, torch.float32)
    assert torch.equal(e.read(), want[1:3])


@gpu
def test_sizes_past_32_bits_are_refused():
    from graphvae import _hip, ops
    E, dev = _hip.GvaeHipError, "cuda"
    big = 2 ** 32 + 32      # (the C entry points would see 32)
    one = torch.zeros(1, 1, 1, device=dev)
    for shape in [(1, big, 1), (big, 1, 1)]:
        with pytest.raises(E):
            ops.group_norm_act(one.expand(shape), None, None, 1)
        with pytest.raises(E):
            st = torch.zeros(1, 1, device=dev)
            ops.group_norm_act_backward(one.expand(shape), one.expand(shape), None, None, st, st, 1)
    x = torch.empty(1, big, dtype=torch.float16, device=dev)
    with pytest.raises(E):
        ops.checkpoint8(x)
    c = ops.Checkpoint8(torch.empty(1, 16, dtype=torch.int8, device=dev), torch.empty(1, 1, dtype=torch.uint8, device=dev), 8)
    with pytest.raises(E):
        ops.linear_wgrad8(x, c)
    del x
    c = ops.Checkpoint8(torch.empty(1, big, dtype=torch.int8, device=dev),
                        torch.empty(1, big // 32, dtype=torch.uint8, device=dev), big)
    with pytest.raises(E):
        c.read()


@gpu
def test_two_graphs_and_two_streams_at_once():
    """Two captured layers replayed on two streams beside each other, and eager layers on both: as each alone."""
    from graphvae import ops
    sets = [_layer_inputs(torch.bfloat16, 11, B=40, N=150, I=64, O=192), _layer_inputs(torch.float32, 12)]
    alone = [_layer(ops, *s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_layer(ops, *s))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for t in [t for out in outs for t in out]:
            t.zero_()
        torch.cuda.synchronize()
        eager = []
        for _ in range(4):
            for graph, stream, s in zip(graphs, streams, sets):
                with torch.cuda.stream(stream):
                    graph.replay()
                    eager.append(_layer(ops, *s))
        torch.cuda.synchronize()
        for k, want in enumerate(alone):
            assert all(torch.equal(p, q) for got in [outs[k], *eager[k::2]] for p, q in zip(got, want))


@gpu
@pytest.mark.parametrize("shape", [(2, 2 ** 21, 520, 4), (70000, 64, 512, 4)])
def test_group_norm_past_32_bit_offsets(shape):
    """A graph of rows that repeat a pattern has the pattern's statistics, values and dx: the last rows of more
    than 2^31 values against the pattern alone, within its rounding and that of the sums' other order."""
    from graphvae import ops
    B, N, C, G = shape
    n = min(N, 1024)
    g = torch.Generator(device="cuda").manual_seed(5)
    base, dbase = (torch.randn(n, C, generator=g, device="cuda").half() for _ in range(2))
    w, b = torch.randn(C, generator=g, device="cuda"), torch.randn(C, generator=g, device="cuda")
    x, dy = (t.expand(B, N // n, n, C).reshape(B, N, C).contiguous() for t in (base, dbase))
    assert x.numel() > 2 ** 31
    one, done = base[None], dbase[None]
    r, e = (ops.group_norm_act(t, w, b, G, act="silu") for t in (x, one))
    # (values of a few units: two of their last places of half, and 2^-16 for sums of up to 2^28 values)
    assert ((r.mean - e.mean).abs() <= 2.0 ** -16).all() and ((r.rstd / e.rstd - 1).abs() <= 2.0 ** -16).all()
    for got in (r.y[-1, -n:], r.y[0, :n]):
        assert ((got.float() - e.y[0].float()).abs() <= 2.0 ** -10 * (e.y[0].float().abs() + 2.0 ** -4)).all()
    keep = ops.checkpoint8(x)
    del r
    for src, osrc in ((x, one), (keep, ops.checkpoint8(one))):
        d = ops.group_norm_act_backward(dy, src, w, b, e.mean.expand(B, G).contiguous(),
                                        e.rstd.expand(B, G).contiguous(), G, act="silu")
        f = ops.group_norm_act_backward(done, osrc, w, b, e.mean, e.rstd, G, act="silu")
        for got in (d[0][-1, -n:], d[0][0, :n]):
            assert ((got.float() - f[0][0].float()).abs() <= 2.0 ** -10 * (f[0][0].float().abs() + 2.0 ** -4)).all()
        for k in (1, 2):
            want = f[k].double() * (B * (N // n))
            assert ((d[k].double() - want).abs() <= 2.0 ** -12 * want.abs().max()).all()
        del d


@gpu
def test_wgrad_past_32_bit_offsets():
    """More than 2^31 gradients and codes; all but the last rows of the gradient are 0: exact."""
    from graphvae import ops
    M, O, I = 2 ** 21 + 77, 1030, 1040
    g = torch.Generator(device="cuda").manual_seed(6)
    dy = torch.zeros(M, O, dtype=torch.float16, device="cuda")
    codes = torch.zeros(M, I, dtype=torch.int8, device="cuda")
    codes[-300:] = torch.randint(-127, 128, (300, I), generator=g, device="cuda").to(torch.int8)
    codes[:300] = 1
    dy[-300:] = torch.randint(-1, 2, (300, O), generator=g, device="cuda").half()
    assert dy.numel() > 2 ** 31 and codes.numel() > 2 ** 31
    c = ops.Checkpoint8(codes, torch.full((M, -(-I // 32)), 127, dtype=torch.uint8, device="cuda"), I)
    dw, db = ops.linear_wgrad8(dy, c)
    # (sums of 300 products of at most 127: integers under 2^16, exact in fp32; half rounds them once)
    want = (dy[-300:].double().t() @ codes[-300:].double()).float().half()
    assert torch.equal(dw, want) and torch.equal(db, dy[-300:].double().sum(0).float().half())
