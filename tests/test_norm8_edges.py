"""Group norm, 8-bit checkpoints and weight gradients where values, sizes or callers are at an edge: what is
not finite stays where it belongs, extreme but finite values, the precision of the activations.  Bounds as
in test_norm8.py: u = 2^-24 for every fp32 operation, half a step of the type for the result."""
import pytest
import torch

from test_norm8 import (ACTS, DEPTH, DTYPES, U32, act_ref, bwd_ref, half_step, make_x, norm_ref, per_channel, slope_ref,
                        subnormal)

gpu = pytest.mark.gpu

# (rows, channels, groups): a last block of 32 channels that is not full, in the resident form (a slab of the whole row,
# lanes behind the last channel) and in the split form
RAGGED_BLOCKS = [(10, 40, 5), (20, 40, 2), (20, 45, 9), (20, 48, 8), (10, 100, 5), (7, 33, 3), (6000, 40, 5),
                 (9000, 45, 9)]


# ------------------------------------------------------------------ what is not finite
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", RAGGED_BLOCKS)
def test_output_checkpoint_beside_a_group_that_is_not_finite(dtype, shape):
    """An infinity or a NaN in the first group reaches the blocks of that group's channels and no other: the
    output's checkpoint is the one that checkpoint8 makes of the output, in the row's last block too."""
    from graphvae import ops
    N, C, G = shape
    x, w, b, _, _ = make_x(2, N, C, dtype, 21)
    first, blocks = C // G, -(-C // 32)
    touched = -(-first // 32)
    for k, act in enumerate(ACTS):
        bad = x.clone()
        bad[1, N // 2, first // 2] = (float("nan"), float("inf"), float("-inf"), float("nan"))[k]
        r = ops.group_norm_act(bad.cuda(), w.cuda(), b.cuda(), G, act=act, keep_x=True, keep_y=True)
        assert r.y[1, :, first:].isfinite().all() and r.y[0].isfinite().all()
        for got, src in ((r.y8, r.y), (r.x8, bad.cuda())):
            want = ops.checkpoint8(src)
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales), act
        assert (r.y8.scales[1, :, :touched] == 255).all() or act != "none"
        assert (r.y8.scales[1, :, touched:blocks] != 255).all() and (r.y8.scales[0] != 255).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C,G,which", [(40, 5, 0), (42, 21, 0), (42, 21, 20), (33, 33, 32)])
def test_output_checkpoint_beside_a_large_constant_group(dtype, C, G, which):
    """A group of equal values of 2^120: its mean is exact (8 rows and a power of two of channels), its
    variance 0, its output act(bias), and the output's checkpoint is that of the output."""
    from graphvae import ops
    x, w, b, _, _ = make_x(2, 8, C, dtype, 22)
    n = C // G
    x[1, :, which * n:(which + 1) * n] = 2.0 ** 120
    for act in ACTS:
        r = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act=act, keep_y=True)
        assert r.mean[1, which].item() == 2.0 ** 120 and r.y.isfinite().all()
        want = ops.checkpoint8(r.y)
        assert torch.equal(r.y8.codes, want.codes) and torch.equal(r.y8.scales, want.scales), act
        assert (r.y8.scales != 255).all()


# ------------------------------------------------------------------ extreme but finite values
@gpu
@pytest.mark.parametrize("dtype,spread", [(torch.float32, 1e17), (torch.bfloat16, 3e17)])
@pytest.mark.parametrize("shape", [(2, 3000, 32, 2), (1, 20000, 24, 3), (2, 5000, 33, 11)])
def test_split_statistics_of_means_whose_squares_overflow(dtype, spread, shape):
    """Means of 4e19 (squared: over the largest fp32) with deviations whose squares are not: finite, and within
    the bounds of any other mean."""
    from graphvae import ops
    B, N, C, G = shape
    g = torch.Generator().manual_seed(23)
    sign = 1.0 - 2.0 * (torch.arange(C) // (C // G) % 2)
    x = (4e19 * sign + spread * torch.randn(B, N, C, generator=g)).to(dtype)
    _, w, b, rows, _ = make_x(B, N, C, dtype, 23)
    rows[0] = N
    x = torch.where(torch.arange(N)[None, :, None] < rows[:, None, None], x, torch.zeros_like(x))
    r = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act="none", rows=rows.cuda())
    y, mean, rstd, tol, dmean, drel = norm_ref(x, w, b, G, "none", 1e-5, rows)
    assert ((r.mean.cpu().double() - mean).abs() <= dmean + 2 * U32 * mean.abs()).all()
    assert ((r.rstd.cpu().double() / rstd - 1).abs() <= drel + 4 * U32).all()
    assert ((r.y.cpu().double() - y).abs() <= half_step(dtype) * y.abs() + 1.01 * tol + subnormal(dtype)).all()


def _far(B, N, C, dtype):
    """Values of 1024 and, one in a hundred, the next one of the type (fp32: 1025): 10^3 to 10^4 deviations from 0."""
    g = torch.Generator().manual_seed(24)
    step = {torch.float32: 1.0, torch.bfloat16: 8.0, torch.float16: 1.0}[dtype]
    x = (1024.0 + step * (torch.rand(B, N, C, generator=g) < 0.01)).to(dtype)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    dy = (0.5 + torch.rand(B, N, C, generator=g)).to(dtype)
    return x, w, b, dy


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 40, 48, 6), (2, 4000, 48, 6), (2, 6000, 45, 9)])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_values_far_from_zero_keep_their_bits(dtype, shape, act):
    """With the mean and rstd that are used (fp32), x - mean is off by u of itself only, however far from zero
    both lie, in the resident and in the split form alike."""
    from graphvae import ops
    B, N, C, G = shape
    x, w, b, dy = _far(B, N, C, dtype)
    r = ops.group_norm_act(x.cuda(), w.cuda(), b.cuda(), G, act=act)
    m, rs = (per_channel(t.cpu().double(), C) for t in (r.mean, r.rstd))
    h = (x.double() - m) * rs
    z = h * w.double() + b.double()
    # x - mean, its product with rstd (or rstd's with w) and that with w: u each; the sum: u of it
    ez = 3 * U32 * (h * w).abs() + U32 * z.abs()
    ry = act_ref(z, act)
    tol = 1.13 * ez + (12 * U32 * z.abs() if act != "none" else 0.0)
    err = (r.y.cpu().double() - ry).abs()
    assert (err <= half_step(dtype) * ry.abs() + 1.01 * tol + subnormal(dtype)).all()
    _, dw, db = ops.group_norm_act_backward(dy.cuda(), x.cuda(), w.cuda(), b.cuda(), r.mean, r.rstd, G, act=act)
    dz = dy.double() * slope_ref(z, act)
    edz = dy.double() * (1.2 * ez + 16 * U32) if act != "none" else 0.0 * dz
    # two roundings of h and DEPTH of the sums (with 80 more over graphs and chunks)
    edw = (edz * h.abs() + (3 + DEPTH + 80) * U32 * (dz * h).abs()).sum((0, 1))
    edb = (edz + (DEPTH + 80) * U32 * dz.abs()).sum((0, 1))
    assert ((dw.cpu().double() - (dz * h).sum((0, 1))).abs() <= 1.01 * edw).all()
    assert ((db.cpu().double() - dz.sum((0, 1))).abs() <= 1.01 * edb).all()


@gpu
def test_large_constant_rows_in_both_forms():
    """bf16 rows of one value whose product with 1 / sqrt(eps) is over the largest fp32 (sums of it are not, and
    with powers of two all round): the norm's value is 0, y the bias."""
    from graphvae import ops
    for N in (8, 16384):
        x = torch.full((1, N, 8), 2.0 ** 100, dtype=torch.bfloat16, device="cuda")
        x[:, :, 4:] = -2.0 ** 105
        b = torch.arange(8, dtype=torch.float32, device="cuda")
        r = ops.group_norm_act(x, None, b, 2, act="none", eps=1e-24)
        assert torch.equal(r.y.float(), b.expand(1, N, 8))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 40, 48, 6), (2, 4000, 48, 6), (2, 6000, 45, 9)])
@pytest.mark.parametrize("scale", [2.0 ** -62, 2.0 ** 60])
def test_gradients_of_very_small_and_very_large_values(dtype, shape, scale):
    """The norm does not depend on the scale of its input: with mean and rstd to match, gradients times 2^12 of
    values of 2^-62 and 2^60 stay within the bounds of ordinary ones."""
    from graphvae import ops
    B, N, C, G = shape
    x, w, b, rows, dy = make_x(B, N, C, dtype, 31)
    x, dy = x * scale, dy * 2.0 ** 12
    x = torch.where(torch.arange(N)[None, :, None] < rows[:, None, None], x, torch.zeros_like(x))
    g = torch.Generator().manual_seed(32)
    mean, rstd = 0.3 * torch.randn(B, G, generator=g) * scale, (0.5 + torch.rand(B, G, generator=g)) / scale
    for act in ("none", "silu"):
        got = ops.group_norm_act_backward(dy.cuda(), x.cuda(), w.cuda(), b.cuda(), mean.cuda(), rstd.cuda(), G, act=act,
                                          rows=rows.cuda())
        dx, dw, db, edx, edw, edb = bwd_ref(dy, x, w, b, mean, rstd, G, act, rows)
        assert ((got[0].cpu().double() - dx).abs() <= half_step(dtype) * dx.abs() + 1.01 * edx + subnormal(dtype)).all()
        assert ((got[1].cpu().double() - dw).abs() <= 2 * edw).all()
        assert ((got[2].cpu().double() - db).abs() <= 2 * edb).all()


# ------------------------------------------------------------------ activations
@gpu
@pytest.mark.parametrize("N", [1, 20000])
@pytest.mark.parametrize("lo,hi", [(-4.0, -2.0), (-6.0, 6.0), (-1.0, 1.0)])
def test_gelu_in_fp32_has_the_precision_of_its_plain_form(N, lo, hi):
    """GELU and its slope alone (weight 0, so that z is the bias; one live row, so that dbias is the slope): the
    root mean square of their error against 64 bits is at most 1.5 times that of z (1 + erf(z / sqrt 2)) / 2 and its
    slope evaluated in fp32 operation by operation.  N: resident and split form."""
    from graphvae import ops
    C = 4096
    z = lo + (hi - lo) * torch.rand(C, generator=torch.Generator().manual_seed(25))
    x = torch.randn(1, 1, C, generator=torch.Generator().manual_seed(26)).expand(1, N, C).cuda()
    rows = torch.ones(1, dtype=torch.int32, device="cuda")
    zero, bias = torch.zeros(C, device="cuda"), z.cuda()
    r = ops.group_norm_act(x, zero, bias, 1, act="gelu", rows=rows)
    _, _, db = ops.group_norm_act_backward(torch.ones_like(x[:, :1]).expand(1, N, C), x, zero, bias, r.mean, r.rstd, 1,
                                           act="gelu", rows=rows)
    cdf = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
    plain = (z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2.0 * torch.pi) ** -0.5)
    for got, form, want in zip((r.y[0, 0], db), plain, (act_ref(z.double(), "gelu"), slope_ref(z.double(), "gelu"))):
        rms = [float((t.cpu().double() - want).square().mean().sqrt()) for t in (got, form)]
        assert 0.0 < rms[0] <= 1.5 * rms[1], rms


# ------------------------------------------------------------------ autograd
def test_inputs_that_require_grad_are_refused():
    """While grad mode is on; with it off the same calls get as far as asking for a device."""
    from graphvae import _hip, ops
    x, g, w = torch.zeros(2, 4, 32), torch.zeros(2, 4, 32), torch.ones(32)
    st = torch.zeros(2, 4)
    c = ops.Checkpoint8(torch.zeros(2, 4, 32, dtype=torch.int8), torch.zeros(2, 4, 1, dtype=torch.uint8), 32)

    def calls(x, g, w, b):
        return [lambda: ops.group_norm_act(x, w, b, 4), lambda: ops.group_norm_act_backward(g, x, w, b, st, st, 4)]

    for k in range(4):
        args = [x, g, w, w.clone()]
        args[k] = args[k].clone().requires_grad_()
        for n, call in enumerate(calls(*args)):
            unused = (n, k) == (0, 1)      # (the forward takes no gradient)
            with pytest.raises(_hip.GvaeHipError, match="expected a device tensor" if unused else "requires grad"):
                call()
            with torch.no_grad(), pytest.raises(_hip.GvaeHipError, match="expected a device tensor"):
                call()
    lone = [lambda t: ops.checkpoint8(t), lambda t: ops.linear_wgrad8(t, c),
            lambda t: ops.group_norm_act_backward(t, c, w, None, st, st, 4)]
    for call in lone:
        with pytest.raises(_hip.GvaeHipError, match="requires grad"):
            call(x.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(_hip.GvaeHipError, match="expected a device tensor"):
            call(x.clone().requires_grad_())
        with pytest.raises(_hip.GvaeHipError, match="expected a device tensor"):
            call(x)


class _NormFunction(torch.autograd.Function):
    """The operators in an autograd node, the input kept in 8 bits."""

    @staticmethod
    def forward(ctx, x, w, b):
        from graphvae import ops
        r = ops.group_norm_act(x, w, b, 4, act="silu", keep_x=True)
        ctx.kept, ctx.args = r.x8, (w, b, r.mean, r.rstd)
        return r.y

    @staticmethod
    def backward(ctx, dy):
        from graphvae import ops
        # (the gradient of a sum is one value expanded along all axes; channels have to be contiguous)
        return ops.group_norm_act_backward(dy.contiguous(), ctx.kept, *ctx.args, 4, act="silu")


@gpu
def test_operators_in_an_autograd_function():
    """Leaves that require grad, through a Function: the gradients of the plain calls, bit for bit."""
    from graphvae import ops
    g = torch.Generator(device="cuda").manual_seed(27)
    leaves = [torch.randn(s, generator=g, device="cuda").requires_grad_() for s in ((3, 20, 48), (48,), (48,))]
    y = _NormFunction.apply(*leaves)
    y.sum().backward()
    x, w, b = (t.detach() for t in leaves)
    r = ops.group_norm_act(x, w, b, 4, act="silu", keep_x=True)
    want = ops.group_norm_act_backward(torch.ones_like(x), r.x8, w, b, r.mean, r.rstd, 4, act="silu")
    assert torch.equal(y.detach(), r.y) and all(torch.equal(t.grad, e) for t, e in zip(leaves, want))


# ------------------------------------------------------------------ weight gradients of the smallest gradients
@gpu
@pytest.mark.parametrize("dtype,exponent", [(torch.float32, -110), (torch.float32, -103), (torch.bfloat16, -133),
                                            (torch.bfloat16, -126), (torch.float16, -24), (torch.float16, -15)])
def test_wgrad_of_small_gradients(dtype, exponent):
    """One row, one power of two as input: dW is the gradient times it, exactly, down to where the last piece
    of a gradient is the smallest bf16 number, 2^-133: |dy| >= 2^-110 in fp32, every value of bf16 and half."""
    from graphvae import ops
    g = torch.Generator().manual_seed(28)
    dy = (2.0 ** exponent * (1 + torch.rand(1, 200, generator=g, dtype=torch.float64))).to(dtype)
    dy[0, ::3] *= -1
    up = 60 if dtype != torch.float16 else 8
    c = ops.checkpoint8(torch.full((1, 40), 2.0 ** up).cuda())
    dw, db = ops.linear_wgrad8(dy.cuda(), c)
    want = (dy.double() * 2.0 ** up).t().expand(200, 40).to(dtype)
    assert torch.equal(dw.cpu(), want) and torch.equal(db.cpu(), dy[0]) and dy.all()


@gpu
def test_wgrad_below_the_smallest_piece():
    """fp32 gradients under 2^-110: what lies below 2^-133 is dropped, and no more."""
    from graphvae import ops
    g = torch.Generator().manual_seed(29)
    dy = (torch.randn(1, 300, generator=g) * torch.exp2(-torch.randint(110, 136, (1, 300), generator=g).float())).float()
    c = ops.checkpoint8(torch.full((1, 40), 2.0 ** 60).cuda())
    dw, db = ops.linear_wgrad8(dy.cuda(), c)
    want = (dy.double() * 2.0 ** 60).t().expand(300, 40)
    assert ((dw.cpu().double() - want).abs() < 2.0 ** (60 - 133)).all() and torch.equal(db.cpu(), dy[0])
