"""The 8-bit product, its quantiser and the Newton-Schulz orthogonalisation against plain 64-bit forms.

quantize_i8  equal to its definition, formed here in numpy's float32 (IEEE division, round half to even).
gemm_i8      the integer sums are exact; scale_a, scale_b, alpha and the conversion of the sum each round once in float
             (u = 2^-24), beta * C is fused, the result rounds once to C's type (half a step, u_T):
                 |C - exact| <= 4 u |alpha S sa sb| + (u + u_T) |exact| + the smallest subnormal of the type.
newton_schulz  in the 2-norm (Frobenius) against 64 bits, by emulations in 64 bits that disturb every stored matrix (X, S, B of
             each step) by independent relative errors, uniform up to the size that one store makes: half a step of
             float16 (2^-11) for bfloat16; for float and float16 2^-22 per stored pair plus the float accumulation of a
             k-long sum (k/16 additions of one half-step 2^-24 each, three products).  With r the root mean square of the
             emulations' errors the allowed error is sqrt(9 steps) r, and half a step for Y.  To first order the error is a sum
             of one term per stored matrix, 3 steps of them.  A store's true error is at most sqrt(3) times the uniform
             one's root mean square, and n terms of mean squares e_j^2 add up to at most sqrt(n) sqrt(sum e_j^2)
             (Cauchy-Schwarz), when all of them point the same way, as they can in a 1 x 1 matrix: sqrt(3 steps) sqrt(3) r."""
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

QUINTIC = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {k: torch.finfo(t).eps / 2 for k, t in TYPES.items()}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


@pytest.fixture(scope="module")
def bl(lib):
    if not torch.cuda.is_available():
        pytest.fail("marked gpu but no CUDA device is visible")
    import batchlas_b200
    yield batchlas_b200
    assert batchlas_b200.device_status() == 0


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def placed(x, pad=0, gap=0, offset=0, fill=7):
    """The values of x (batch, cols, rows) on the GPU with ld = rows + pad, `gap` elements between items and `offset` before the
    first; returns the view and the whole buffer."""
    b, c, r = x.shape
    stride = c * (r + pad) + gap
    back = torch.full((offset + b * stride,), fill, dtype=x.dtype, device="cuda")
    view = back[offset:].as_strided((b, c, r), (stride, r + pad, 1), offset)
    view.copy_(x)
    return view, back


# ---- quantize_i8 ------------------------------------------------------------------------------------------------------------
def quantize_reference(x):
    """x: float32 numpy (batch, cols, k)."""
    top = np.max(np.abs(x), axis=-1) if x.shape[-1] else np.zeros(x.shape[:-1], np.float32)
    scale = (top * (np.float32(1) / np.float32(127))).astype(np.float32)
    usable = (scale > 0) & np.isfinite(scale)
    with np.errstate(all="ignore"):
        q = np.rint((x / np.where(usable, scale, np.float32(1))[..., None]).astype(np.float32))
    return np.where(usable[..., None], np.clip(q, -127, 127), 0).astype(np.int8), scale


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("batch,cols,k", [(1, 1, 1), (1, 1, 16), (2, 3, 7), (1, 5, 33), (3, 17, 130), (1, 2, 4096), (2, 9, 1001),
                                          (1, 1, 20000), (1, 700, 64), (1, 3, 70001), (70000, 1, 3), (2, 33, 2048)])
def test_quantize(bl, kind, batch, cols, k):
    x = (torch.randn(batch, cols, k, generator=gen(k + cols)) * torch.exp(3 * torch.randn(batch, cols, 1, generator=gen(k)))).to(TYPES[kind])
    x[0, 0, : k // 3] = x[0, 0].abs().max() / 2   # a tie: 63.5 steps
    for pad, gap, offset in [(0, 0, 0), (3, 5, 1), (16, 0, 8)]:
        view, _ = placed(x, pad, gap, offset)
        q, qb = placed(torch.zeros(batch, cols, k, dtype=torch.int8), pad, gap, offset)
        s = torch.empty(batch, cols, device="cuda")
        bl.quantize_i8(view, q, s)
        want_q, want_s = quantize_reference(x.float().numpy())
        assert np.array_equal(s.cpu().numpy(), want_s)
        assert np.array_equal(q.cpu().numpy(), want_q)
        q.fill_(7)
        assert bool((qb == 7).all()), "padding was written"


@pytest.mark.parametrize("kind,bits", [("bf16", 8), ("f16", 11)])
def test_quantize_every_halfway_point_of_the_half_types(bl, kind, bits):
    """Every mantissa as the column's largest value, every mantissa below it in nine binades as an element."""
    mantissas = np.arange(2 ** (bits - 1), 2 ** bits, dtype=np.float32) / 2 ** bits
    values = (mantissas[:, None] * np.exp2(-np.arange(9, dtype=np.float32))).ravel()
    for first in range(0, len(mantissas), 128):
        tops = mantissas[first:first + 128, None]
        x = np.where(values <= tops, values, 0)
        x[:, ::2] *= -1
        x[:, 0] = tops[:, 0]
        d = torch.from_numpy(x.astype(np.float32))[None].to(TYPES[kind])
        q, s = bl.quantize_i8(d.cuda())
        want_q, want_s = quantize_reference(d.float().numpy())
        assert np.array_equal(s.cpu().numpy(), want_s) and np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("kind", TYPES)
def test_quantize_special_columns(bl, kind):
    t = TYPES[kind]
    x = torch.randn(1, 9, 50, generator=gen(3)).to(t)
    x[0, 0] = 0
    x[0, 1, 7] = float("inf")
    x[0, 2, 49] = float("nan")
    x[0, 3, 0] = -float("inf")
    x[0, 3, 1] = float("nan")
    x[0, 4] = 0
    x[0, 4, 3] = torch.finfo(t).smallest_normal * torch.finfo(t).eps   # the smallest subnormal
    x[0, 5] = torch.finfo(t).max * torch.sign(x[0, 5].float()).to(t)
    x[0, 6] = -0.0
    q, s = bl.quantize_i8(x.cuda())
    want_q, want_s = quantize_reference(x.float().numpy())
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True) and np.isnan(want_s[0, 2]) and np.isinf(want_s[0, 1])
    assert np.array_equal(q.cpu().numpy(), want_q)


def test_quantize_empty_columns(bl):
    q, s = bl.quantize_i8(torch.empty(2, 3, 0, device="cuda"))
    assert q.shape == (2, 3, 0) and bool((s == 0).all())
    q, s = bl.quantize_i8(torch.empty(2, 0, 5, device="cuda"))
    assert s.shape == (2, 0)


# ---- gemm_i8 ----------------------------------------------------------------------------------------------------------------
def gemm_i8_check(got, kind, a, b, sa, sb, alpha, beta, prior):
    f = lambda t: t.double().cpu()  # noqa: E731
    total = torch.matmul(f(b), f(a).transpose(-2, -1))      # exact: below 2^53
    scaled = alpha * total * (1 if sa is None else f(sa).unsqueeze(-2)) * (1 if sb is None else f(sb).unsqueeze(-1))
    want = scaled + (beta * f(prior) if beta != 0 else 0)
    u = 2.0 ** -24
    allowed = 4 * u * scaled.abs() + (u + HALF_STEP[kind]) * want.abs() + TINY[kind]
    over = (f(got) - want).abs() - allowed
    assert bool((over <= 0).all()), (float(over.max()), bl_name())


def bl_name():
    import batchlas_b200
    return batchlas_b200.last_kernel_name()


SHAPES = [(1, 1, 1, 1), (1, 1, 16, 3), (7, 5, 3, 2), (16, 1, 32, 1), (128, 1, 256, 1), (129, 17, 130, 2), (256, 16, 4096, 1),
          (512, 33, 2048, 2), (300, 257, 1000, 1), (64, 500, 48, 2), (640, 384, 512, 1), (1000, 96, 128, 5), (40, 8, 8192, 1), (200, 32, 1040, 2), (17, 24, 190, 3),
          (2048, 3, 400, 1), (257, 1024, 272, 1), (128, 128, 16, 2), (1, 700, 640, 1), (700, 1, 640, 1), (513, 130, 96, 3), (2305, 2300, 160, 1),
          (500, 300, 272, 20)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k,batch", SHAPES, ids=str)
def test_gemm_i8(bl, kind, m, n, k, batch):
    g = gen(m + 3 * n + 7 * k)
    a = torch.randint(-128, 128, (batch, m, k), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (batch, n, k), generator=g, dtype=torch.int8)
    sa, sb = torch.rand(batch, m, generator=g) * 1e-2, torch.randn(batch, n, generator=g) * 1e-2
    c0 = torch.randn(batch, n, m, generator=g).to(TYPES[kind])
    k16 = (-k) % 16
    # packed; ld and stride multiples of 16 bytes off packed ones; nothing aligned
    for pad, gap, offset, alpha, beta in [(0, 0, 0, 1.0, 0.0), (k16 + 16, 48, 32, -0.75, 0.5), (1, 3, 1, 1.0, 1.0)]:
        va, _ = placed(a, pad, gap, offset)
        vb, _ = placed(b, pad, gap, offset)
        cin = c0.clone()
        if beta == 0:
            cin[:] = float("nan")                           # never read then
        vc, cb = placed(cin, pad, gap, offset)
        bl.gemm_i8(va, vb, vc, sa.cuda(), sb.cuda(), alpha, beta)
        gemm_i8_check(vc, kind, a, b, sa, sb, alpha, beta, c0)
        vc.fill_(7)
        assert bool((cb == 7).all()), "padding of C was written"


def test_gemm_i8_scales_and_broadcast(bl):
    g = gen(5)
    m, n, k, batch = 96, 40, 160, 6
    a = torch.randint(-128, 128, (1, m, k), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (batch, n, k), generator=g, dtype=torch.int8)
    sa, sb = torch.rand(m, generator=g), torch.rand(batch, n, generator=g)
    for ua, ub in [(sa, sb), (None, sb), (sa, None), (None, None)]:
        c = torch.empty(batch, n, m, device="cuda")
        bl.gemm_i8(a.cuda(), b.cuda(), c, None if ua is None else ua.cuda(), None if ub is None else ub.cuda())
        gemm_i8_check(c, "f32", a.expand(batch, m, k), b, None if ua is None else ua.expand(batch, m), ub, 1.0, 0.0, c)
    # items of C interleaved inside the leading dimension (heads side by side in one row)
    wide = torch.full((n, batch, m), 7.0, device="cuda")
    bl.gemm_i8(a.cuda(), b.cuda(), wide.permute(1, 0, 2), sa.cuda(), sb.cuda())
    gemm_i8_check(wide.permute(1, 0, 2), "f32", a.expand(batch, m, k), b, sa.expand(batch, m), sb, 1.0, 0.0, wide)


@pytest.mark.parametrize("n", [1, 9, 200])
def test_gemm_i8_largest_sums_and_non_finite_scales(bl, n):
    k, m = 131071, 130
    a = torch.full((1, m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((1, n, k), -128, dtype=torch.int8, device="cuda")
    b[0, -1] = 127
    for pad in (0, 1):   # 131071 is odd: pad 1 makes the columns 16-byte aligned
        va = torch.nn.functional.pad(a, (0, pad))[:, :, :k]
        vb = torch.nn.functional.pad(b, (0, pad))[:, :, :k]
        c = torch.empty(1, n, m, device="cuda")
        bl.gemm_i8(va, vb, c)
        want = torch.full((1, n, m), 128.0 * 128 * k, dtype=torch.float64)
        want[0, -1] = -128.0 * 127 * k
        assert torch.equal(c.cpu(), want.float())
    sb = torch.ones(1, n, device="cuda")
    sb[0, -1] = float("nan")
    c = torch.empty(1, n, m, device="cuda", dtype=torch.bfloat16)
    bl.gemm_i8(a[:, :, :64].contiguous(), b[:, :, :64].contiguous(), c, None, sb)
    assert bool(c[0, -1].isnan().all()) and not bool(c[0, :-1].isnan().any())


def test_gemm_i8_empty_sums(bl):
    c = torch.full((2, 3, 5), 2.0, device="cuda")
    e = torch.empty(2, 5, 0, dtype=torch.int8, device="cuda")
    bl.gemm_i8(e, torch.empty(2, 3, 0, dtype=torch.int8, device="cuda"), c, torch.full((5,), float("nan"), device="cuda"), None, 1.0, 0.5)
    assert bool((c == 1).all())
    bl.gemm_i8(torch.empty(2, 0, 8, dtype=torch.int8, device="cuda"), torch.zeros(2, 3, 8, dtype=torch.int8, device="cuda"),
               torch.empty(2, 3, 0, device="cuda"))


def test_refusals_of_the_python_layer(bl):
    q = torch.zeros(2, 4, 16, dtype=torch.int8, device="cuda")
    c = torch.zeros(2, 4, 4, device="cuda")
    one = torch.ones(4, device="cuda")
    with pytest.raises(RuntimeError, match="incompatible"):
        bl.gemm_i8(q, q[:, :, :8], c)
    with pytest.raises(RuntimeError, match="incompatible"):
        bl.gemm_i8(q, q, c, one[:3])
    with pytest.raises(RuntimeError, match="incompatible"):
        bl.gemm_i8(torch.cat([q, q]), q, c)
    with pytest.raises(TypeError):
        bl.gemm_i8(q, q, c.double())
    with pytest.raises(TypeError):
        bl.gemm_i8(q.float(), q, c)
    with pytest.raises(TypeError):
        bl.gemm_i8(q, q, c, one.double())
    with pytest.raises(ValueError):
        bl.gemm_i8(q, q, c, transA=bl.Transpose.NoTrans)
    with pytest.raises(ValueError):
        bl.gemm_i8(q.transpose(1, 2), q, c)
    with pytest.raises(bl.BlasError):
        bl.gemm_i8(q, q, c[:1].expand(2, 4, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        bl.gemm_i8(q, q.cpu(), c)
    with pytest.raises(TypeError):
        bl.quantize_i8(q)
    with pytest.raises(RuntimeError, match="incompatible"):
        bl.quantize_i8(c, q)
    with pytest.raises(RuntimeError, match="incompatible"):
        bl.quantize_i8(c, scale=one)
    with pytest.raises(TypeError):
        bl.newton_schulz(c.double())
    with pytest.raises(RuntimeError, match="incompatible"):
        bl.newton_schulz(c, c[:, :2])
    with pytest.raises(ValueError):
        bl.newton_schulz(c, coefficients=[(1, 2, 3), (1, 2, 3)], steps=3)
    with pytest.raises(ValueError):
        bl.newton_schulz(c, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(bl.BlasError):
        bl.newton_schulz(c, coefficients=(50.0, 50.0, 50.0))


# ---- newton_schulz ----------------------------------------------------------------------------------------------------------
def newton_schulz_reference(g, steps, sets, eps, disturb=0.0, seed=0, device="cpu"):
    """64-bit form on (batch, cols, rows); `disturb`: relative size of the error of every stored matrix."""
    noise = torch.Generator(device=device).manual_seed(seed)

    def stored(m):
        if disturb == 0:
            return m
        return m * (1 + disturb * (2 * torch.rand(m.shape, generator=noise, dtype=torch.float64, device=device) - 1))

    x = g.to(device).double()
    x = stored(x / (x.flatten(1).norm(dim=1)[:, None, None] + eps))
    if x.shape[1] > x.shape[2]:
        return newton_schulz_reference(g.transpose(1, 2), steps, sets, eps, disturb, seed, device).transpose(1, 2)
    for i in range(steps):
        a, b, c = sets[i % len(sets)]
        s = stored(x @ x.transpose(1, 2))
        x = stored(a * x + stored(b * s + c * s @ s) @ x)
    return x


def newton_schulz_check(got, g, kind, steps=5, sets=(QUINTIC,), eps=1e-7, device="cpu"):
    want = newton_schulz_reference(g, steps, sets, eps, device=device)
    p, q = sorted(g.shape[1:])
    one_store = 2.0 ** -11 if kind == "bf16" else 2.0 ** -22 + 3 * (q / 16 + 1) * 2.0 ** -24
    errors = torch.stack([newton_schulz_reference(g, steps, sets, eps, one_store, p + q + i, device) - want for i in range(8)])
    rms = errors.square().sum((2, 3)).mean(0).sqrt()
    for i in range(g.shape[0]):
        allowed = (9 * steps) ** 0.5 * float(rms[i]) + HALF_STEP[kind] * float(want[i].norm())
        off = float((got[i].to(device).double() - want[i]).norm())
        assert off <= allowed, (i, off, allowed, float(want[i].norm()), bl_name())


def update_like(batch, cols, rows, seed, kind, size=1e-3):
    g = gen(seed)
    rank = max(1, min(cols, rows) // 8)
    low = torch.randn(batch, cols, rank, generator=g) @ torch.randn(batch, rank, rows, generator=g)
    return (size * (low * rank ** -0.5 + 0.5 * torch.randn(batch, cols, rows, generator=g))).to(TYPES[kind])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("batch,cols,rows", [(1, 1, 1), (2, 1, 40), (2, 40, 1), (3, 7, 5), (2, 16, 16), (1, 33, 65), (5, 64, 64),
                                             (2, 128, 128), (1, 100, 128), (2, 128, 250), (1, 129, 127), (1, 64, 1000), (1, 1000, 64),
                                             (2, 200, 300), (1, 300, 200), (1, 385, 256), (1, 256, 512), (2, 520, 513),
                                             (3, 128, 512), (1, 300, 100), (2, 1000, 120), (1, 77, 1030), (2, 2048, 30), (1, 128, 1500),
                                             (1, 100, 4096), (1, 3000, 128)])
def test_newton_schulz(bl, kind, batch, cols, rows):
    g = update_like(batch, cols, rows, cols + rows, kind)
    for pad, gap, offset in [(0, 0, 0), (3, 5, 1)]:
        view, _ = placed(g, pad, gap, offset)
        out, back = placed(torch.zeros_like(g), pad, gap, offset)
        bl.newton_schulz(view, out)
        newton_schulz_check(out, g, kind)
        assert torch.equal(view.cpu(), g), "the input was written"
        out.fill_(7)
        assert bool((back == 7).all()), "padding was written"


@pytest.mark.parametrize("kind,batch,cols,rows", [("bf16", 1, 1900, 2304), ("bf16", 2, 2111, 1700), ("f16", 1, 1100, 1900), ("f32", 1, 1500, 1333),
                                                  ("f32", 3, 260, 1031), ("bf16", 9, 515, 1030), ("f16", 5, 700, 300),
                                                  ("f32", 40, 128, 1000), ("f16", 30, 1030, 128), ("bf16", 300, 50, 40)])
def test_newton_schulz_many_tiles(bl, kind, batch, cols, rows):
    """Pairs of CTAs, several rounds of tiles, and tiles split over clusters; the 64-bit form runs on the GPU too."""
    g = update_like(batch, cols, rows, cols + rows, kind)
    newton_schulz_check(bl.newton_schulz(g.cuda()), g, kind, device="cuda")


def test_newton_schulz_layouts_of_batches(bl):
    g = update_like(1, 40, 72, 2, "f32")
    y = bl.newton_schulz(g.cuda().expand(3, 40, 72))                     # one matrix for every item
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
    newton_schulz_check(y[:1], g, "f32")
    many = update_like(3, 150, 144, 5, "bf16").cuda()
    side_by_side = torch.full((150, 3, 144), 7.0, dtype=torch.bfloat16, device="cuda")
    out = side_by_side.permute(1, 0, 2)                                  # items interleaved inside the leading dimension
    bl.newton_schulz(many, out)
    assert torch.equal(out, bl.newton_schulz(many))


@pytest.mark.parametrize("kind", TYPES)
def test_newton_schulz_coefficients_steps_and_in_place(bl, kind):
    g = update_like(2, 96, 160, 3, kind)
    cubic = [(1.5, -0.5, 0.0)]
    schedule = [(8.2, -23.5, 17.2), (4.1, -2.9, 0.5), (3.9, -2.9, 0.55), (1.875, -1.25, 0.375)]
    for sets, steps in [([QUINTIC], 1), (cubic, 12), (schedule, 4)]:
        d = g.cuda()
        y = bl.newton_schulz(d, d, steps=steps, coefficients=sets if len(sets) > 1 else sets[0])
        assert y is d
        newton_schulz_check(d, g, kind, steps, sets)


@pytest.mark.parametrize("kind", TYPES)
def test_newton_schulz_range_of_inputs(bl, kind):
    big = {"f32": 1e37, "bf16": 1e37, "f16": 1e3}[kind]
    small = {"f32": 1e-30, "bf16": 1e-30, "f16": 1e-4}[kind]
    for size in (big, small):                       # eps 0: the result does not depend on the size
        g = update_like(2, 48, 72, 9, kind, size)
        newton_schulz_check(bl.newton_schulz(g.cuda(), eps=0.0), g, kind, eps=0.0)
    g = update_like(1, 40, 40, 10, kind, 1e-4)      # eps as large as the norm and larger
    for eps in (1e-3, 0.1):
        newton_schulz_check(bl.newton_schulz(g.cuda(), eps=eps), g, kind, eps=eps)
    z = torch.zeros(2, 40, 30, dtype=TYPES[kind], device="cuda")
    assert bool((bl.newton_schulz(z) == 0).all())
    diagonal = torch.eye(70)[None].to(TYPES[kind])  # one entry per row: the least even distribution
    newton_schulz_check(bl.newton_schulz(diagonal.cuda()), diagonal, kind)
    one = torch.zeros(1, 64, 96, dtype=TYPES[kind])
    one[0, 5, 7] = 3.0
    newton_schulz_check(bl.newton_schulz(one.cuda()), one, kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols,rows", [(64, 96), (300, 260)])
def test_newton_schulz_non_finite_items_stay_apart(bl, kind, cols, rows):
    g = update_like(4, cols, rows, 4, kind)
    g[1, 3, 3] = float("nan")
    g[2, 0, 0] = float("inf")
    y = bl.newton_schulz(g.cuda())
    assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
    newton_schulz_check(y[[0, 3]], g[[0, 3]], kind)


# ---- sizes past 32 bits -----------------------------------------------------------------------------------------------------
def test_quantize_and_product_past_32_bit_offsets(bl):
    k, cols = 40000, 60001                                  # 2.4e9 elements
    x = torch.zeros(cols, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, k, generator=gen(1)).to(torch.bfloat16).cuda()
    q, s = bl.quantize_i8(x)
    want_q, want_s = quantize_reference(x[-3:].float().cpu().numpy())
    assert np.array_equal(q[-3:].cpu().numpy(), want_q) and np.array_equal(s[-3:].cpu().numpy(), want_s)
    assert not bool(s[:-3].any()) and not bool(q[:-3].any())
    del x
    for n in (4, 40):
        b = torch.randint(-128, 128, (n, k), generator=gen(n), dtype=torch.int8).cuda()
        c = bl.gemm_i8(q, b, torch.empty(n, cols, device="cuda"))
        assert torch.equal(c[:, -3:].double(), b.double() @ q[-3:].double().T) and not bool(c[:, :-3].any())
        odd = q.flatten()[1:1 + (cols - 1) * k].view(cols - 1, k)   # the same bytes, every column one byte later
        c = bl.gemm_i8(odd, b, torch.empty(n, cols - 1, device="cuda"))
        assert torch.equal(c[:, -3:].double(), b.double() @ odd[-3:].double().T) and not bool(c[:, :-3].any())


def test_newton_schulz_past_32_bit_offsets(bl):
    """120 x 18 000 001: the iteration is X0 times a polynomial of the 120 x 120 Gram matrix, which 64 bits give exactly enough.
    Three steps of three stores, each off by at most 2^-11 and amplified by at most 3.9 per step that follows, and Y's half step."""
    rows, cols, steps = 120, 18_000_001, 3
    g = torch.empty(cols, rows, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    gram = sum(part.double().T @ part.double() for part in g.split(2_000_000))
    f = float(gram.trace()) ** 0.5 + 1e-7
    one, s = torch.eye(rows, dtype=torch.float64, device="cuda"), gram / f ** 2
    total, (a, b, c) = one, QUINTIC
    for _ in range(steps):
        poly = a * one + b * s + c * s @ s
        total, s = total @ poly, poly @ s @ poly
    y = bl.newton_schulz(g, steps=steps)
    allowed = sum(3 * 2.0 ** -11 * 3.9 ** i for i in range(steps)) + 2.0 ** -8
    for part in (slice(0, 1000), slice(cols // 2, cols // 2 + 1000), slice(cols - 1000, cols)):
        want = g[part].double() / f @ total
        assert float((y[part].double() - want).norm()) <= allowed * float(want.norm())


# ---- together ---------------------------------------------------------------------------------------------------------------
def test_update_quantise_and_serve(bl):
    """A weight takes an orthogonalised update, is quantised by channel and multiplies quantised activations."""
    out_dim, in_dim, tokens = 192, 256, 33
    g = gen(11)
    w = torch.randn(out_dim, in_dim, generator=g) * in_dim ** -0.5
    grad = update_like(1, out_dim, in_dim, 12, "f32")
    x = torch.randn(tokens, in_dim, generator=g).to(torch.bfloat16)
    y = bl.newton_schulz(grad.cuda())
    dw = w.cuda()[None]
    bl.linalg.axpby_into(-0.02, y, 1.0, dw, dw)
    wq, ws = bl.quantize_i8(dw[0])
    xq, xs = bl.quantize_i8(x.cuda())
    out = torch.empty(tokens, out_dim, dtype=torch.bfloat16, device="cuda")
    bl.gemm_i8(wq, xq, out, ws, xs)
    want_q, want_s = quantize_reference(dw.cpu().numpy())
    assert np.array_equal(wq.cpu().numpy(), want_q[0]) and np.array_equal(ws.cpu().numpy(), want_s[0])
    gemm_i8_check(out[None], "bf16", wq[None], xq[None], ws[None], xs[None], 1.0, 0.0, out)
    # against the unquantised layer: each factor is off by at most half a step of its scale
    exact = x.double() @ dw[0].double().cpu().T
    bound = 0.5 * (xs.cpu().double()[:, None] * dw[0].abs().sum(1).cpu().double()
                   + ws.cpu().double() * x.double().abs().sum(1, keepdim=True)
                   + 0.5 * in_dim * xs.cpu().double()[:, None] * ws.cpu().double())
    assert bool(((out.double().cpu() - exact).abs() <= bound * 1.001 + 2.0 ** -8 * exact.abs() + 2.0 ** -8 * bound).all())


def run_all(bl, g, x, w, ws, out, ns, wspace, stream=None):
    bl.newton_schulz(g, ns, workspace=wspace, stream=stream)
    q, s = bl.quantize_i8(x, out["q"], out["s"], stream=stream)
    bl.gemm_i8(w, q, out["y"], ws, s, stream=stream)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_captured_and_replayed_with_new_inputs(bl, kind):
    g, x = update_like(2, 160, 224, 1, kind).cuda(), torch.randn(20, 512, generator=gen(2)).to(TYPES[kind]).cuda()
    w = torch.randint(-127, 128, (300, 512), generator=gen(3), dtype=torch.int8).cuda()
    ws = torch.rand(300, generator=gen(4)).cuda()
    out = {"q": torch.empty(20, 512, dtype=torch.int8, device="cuda"), "s": torch.empty(20, device="cuda"),
           "y": torch.empty(20, 300, dtype=TYPES[kind], device="cuda")}
    ns = torch.empty_like(g)
    space = torch.empty(bl.newton_schulz_workspace_bytes(g), dtype=torch.uint8, device="cuda")
    run_all(bl, g, x, w, ws, out, ns, space)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_all(bl, g, x, w, ws, out, ns, space)
    for seed in (5, 6):
        g.copy_(update_like(2, 160, 224, seed, kind))
        x.copy_(torch.randn(20, 512, generator=gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        replayed = ns.clone(), out["y"].clone()
        ns.zero_(), out["y"].zero_(), space.fill_(0xff)
        run_all(bl, g, x, w, ws, out, ns, space)
        torch.cuda.synchronize()
        assert torch.equal(replayed[0], ns) and torch.equal(replayed[1], out["y"])
        newton_schulz_check(ns, g.cpu(), kind)


def test_two_streams_at_once(bl):
    g = [update_like(1, 256, 384, s, "bf16").cuda() for s in (1, 2)]
    alone = [bl.newton_schulz(x) for x in g]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            outs[i].append(bl.newton_schulz(g[i], stream=s.cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_another_stream_and_its_own_scratch(bl):
    g, x = update_like(1, 300, 200, 1, "f32").cuda(), torch.randn(9, 300, generator=gen(2)).cuda()
    w = torch.randint(-127, 128, (70, 300), generator=gen(3), dtype=torch.int8).cuda()
    want_y, (want_q, want_s) = bl.newton_schulz(g), bl.quantize_i8(x)
    want_c = bl.gemm_i8(w, want_q, torch.empty(9, 70, device="cuda"), None, want_s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    y, q, s, c = torch.zeros_like(want_y), torch.zeros_like(want_q), torch.zeros_like(want_s), torch.zeros_like(want_c)
    torch.cuda.synchronize()
    bl.newton_schulz(g, y, stream=side.cuda_stream)
    bl.quantize_i8(x, q, s, stream=side.cuda_stream)
    bl.gemm_i8(w, q, c, None, s, stream=side.cuda_stream)
    side.synchronize()
    for got, want in ((y, want_y), (q, want_q), (s, want_s), (c, want_c)):
        assert torch.equal(got, want)


FIRST_CALLS_IN_A_CAPTURE = """
import torch, batchlas_b200 as bl
gs = [torch.randn(2, 300, 260, device="cuda"), torch.randn(3, 64, 50, device="cuda").bfloat16()]
ys = [torch.zeros_like(g) for g in gs]
x = torch.randn(40, 512, device="cuda")
w = torch.randint(-127, 128, (96, 512), device="cuda", dtype=torch.int8)
c = torch.zeros(40, 96, device="cuda")
torch.cuda.synchronize()
graphs = []
for i in range(2):                      # two graphs, each with scratch of its own
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1]):
        bl.newton_schulz(gs[i], ys[i])
        q, s = bl.quantize_i8(x)
        bl.gemm_i8(w, q, c, None, s)
for _ in range(3):
    for graph in graphs:
        graph.replay()
torch.cuda.synchronize()
for g, y in zip(gs, ys):
    assert torch.equal(bl.newton_schulz(g), y)
q, s = bl.quantize_i8(x)
assert torch.equal(bl.gemm_i8(w, q, torch.zeros_like(c), None, s), c) and float(c.abs().sum()) > 0
assert bl.device_status() == 0
print("replayed")
"""


def test_first_calls_of_a_process_inside_a_capture(bl):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "replayed" in out.stdout, out.stdout[-2000:] + out.stderr[-2000:]
