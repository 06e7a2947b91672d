"""How close newton_schulz comes to 64 bits, element by element of its arithmetic: every type keeps float accuracy until Y is rounded.

With x the result in 64 bits, rn the rounding to the type and d the error before it, rounding to nearest gives for each element
|rn(x + d) - x| <= |rn(x) - x| + 2 |d|  (rn(x + d) is no further from x + d than rn(x) is), so over any set of elements

    || Y - x || <= || rn(x) - x || + 2 || d ||,

and also <= || d || + u || x || (1 + u) with u half a step of the type.

|| d || comes from emulations in 64 bits of what one store and one product may lose:
  * a stored matrix (X, S, B) is a pair of float16: 2^-22 of each element;
  * the tensor cores drop less than 2^-23 of the running sum at an addition of sixteen products, always towards zero.  Eight such
    additions go to one partial sum (sixteen where a matrix stays in shared memory).  Partial sums are added in float, 2^-24
    each, and the products of two low halves are left out, 2^-22 of each product.
A sum whose terms have one sign grows evenly, so n additions drop less than (1 + 2 + ... + n) / n = (n + 1) / 2 times 2^-23 of it.
These losses go in the same direction everywhere: they are emulated that way, for each of the three products of a step by
itself, and their effects' norms added.  All others, among them n 2^-23 of |sum| + sqrt(sum of squares) (a random walk's size)
for sums with terms of both signs, are drawn independently and uniformly, and twice the root mean square of their effect is allowed.
A single row or column has fewer elements to average over and is allowed three times its share."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

QUINTIC = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIR, HALF = 2.0 ** -22, 2.0 ** -11


@pytest.fixture(scope="module")
def bl(lib):
    if not torch.cuda.is_available():
        pytest.fail("marked gpu but no CUDA device is visible")
    import batchlas_b200
    yield batchlas_b200
    assert batchlas_b200.device_status() == 0


def emulated(g, steps, coefficients, eps, store=0.0, towards_zero=(0.0, 0.0, 0.0), spread=0.0, seed=0):
    """The iteration in 64 bits on (batch, p, q) with p <= q, disturbed as the module's text says."""
    noise = torch.Generator(device=g.device).manual_seed(seed)

    def uniform(m):
        return 2 * torch.rand(m.shape, generator=noise, dtype=torch.float64, device=g.device) - 1

    def stored(m):
        return m * (1 + store * uniform(m)) if store else m

    def product(which, x, y):
        d = x @ y
        out = d * (1 - towards_zero[which]) if towards_zero[which] else d
        if spread:
            rate = spread + (x.shape[-1] / 128 + 1) ** 0.5 * 2.0 ** -24
            out = out + rate * uniform(d) * (d.abs() + (x.square() @ y.square()).sqrt())
        return out

    x = g.double()
    x = stored(x / (x.flatten(1).norm(dim=1)[:, None, None] + eps))
    a, b, c = coefficients
    for _ in range(steps):
        s = stored(product(0, x, x.mT))
        x = stored(a * x + product(2, stored(b * s + c * product(1, s, s)), x))
    return x


def check(got, g, kind, steps=5, coefficients=QUINTIC, eps=1e-7, store=PAIR, additions=None):
    got, g = got.double(), g.to(got.device)
    if g.shape[1] > g.shape[2]:
        got, g = got.mT, g.mT
    want = emulated(g, steps, coefficients, eps)
    if additions is None:
        additions = 16 if g.shape[1] <= 128 and g.shape[2] <= 2048 else 8
    lost, u = (additions + 1) / 2 * 2.0 ** -23, torch.finfo(TYPES[kind]).eps / 2
    same = [emulated(g, steps, coefficients, eps, towards_zero=[lost * (i == j) for j in range(3)]) - want for i in range(3)]
    drawn = [emulated(g, steps, coefficients, eps, store=store, spread=additions * 2.0 ** -23 + 2.0 ** -22, seed=i) - want for i in range(4)]
    rounding = want.to(TYPES[kind]).double() - want
    for dims, share in (((1, 2), 1.0), ((1,), 3.0), ((2,), 3.0)):
        norm = lambda t: t.square().sum(dims).sqrt()  # noqa: E731
        d = sum(norm(e) for e in same) + 2 * torch.stack([norm(e).square() for e in drawn]).mean(0).sqrt()
        allowed, off = torch.minimum(norm(rounding) + 2 * share * d, share * d + u * (1 + u) * norm(want)), norm(got - want)
        over = off / allowed
        assert bool((over <= 1).all()), (dims, float(over.max()), float(off.max()), float(norm(want).max()))


def update_like(batch, cols, rows, seed, kind, size=1e-3):
    g = torch.Generator().manual_seed(seed)
    rank = max(1, min(cols, rows) // 8)
    low = torch.randn(batch, cols, rank, generator=g) @ torch.randn(batch, rank, rows, generator=g)
    return (size * (low * rank ** -0.5 + 0.5 * torch.randn(batch, cols, rows, generator=g))).to(TYPES[kind])


# one CTA, clusters, tiles split over clusters, single tiles and pairs of CTAs, long sums; both orientations
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("batch,cols,rows", [(3, 128, 128), (2, 90, 250), (2, 128, 1500), (1, 2000, 100), (2, 300, 260), (40, 140, 200), (1, 1500, 1333),
                                             (1, 1100, 1900), (1, 160, 40000), (1, 9001, 200)])
def test_float_accuracy_until_the_result_is_rounded(bl, kind, batch, cols, rows):
    g = update_like(batch, cols, rows, cols + rows, kind)
    check(bl.newton_schulz(g.cuda()), g, kind)


@pytest.mark.parametrize("c", [1e-20, -1e-17, 1e-13])
@pytest.mark.parametrize("cols,rows", [(96, 80), (200, 300)])
def test_a_coefficient_next_to_zero(bl, cols, rows, c):
    """A step up to 1.71 before the cubic one, whose largest value then lies inside the interval."""
    g = torch.eye(max(cols, rows))[:cols, :rows].repeat(2, 1, 1) * torch.tensor([1.0, 3e-4])[:, None, None]
    g[1, 0, 0] = 1.0                                    # one singular value near 1, the others small
    y = bl.newton_schulz(g.cuda(), steps=3, coefficients=[(1.7149, 0.0, 0.0), (1.5, -0.5, c), (1.5, -0.5, c)])
    x = g.double().cuda() / (g.double().flatten(1).norm(dim=1)[:, None, None].cuda() + 1e-7)
    d = torch.diagonal(x, dim1=1, dim2=2)
    d = 1.7149 * d
    for _ in range(2):
        d = 1.5 * d - 0.5 * d ** 3 + c * d ** 5
    got = torch.diagonal(y, dim1=1, dim2=2).double()
    # Each stored value is off by at most e of itself (a pair, and a product of sixteen additions, the diagonal having one term).
    # X after the first step: 2 stores of up to 1.7149; the second step's slope there is 1.5 - 1.5 * 1.7149^2 = -2.92, its two terms
    # come to 2.57 and 2.52, from 3 stores; the third step's slope is at most 1.5, its terms below 1 from 3 stores; Y is rounded.
    e = 2.0 ** -22 + 17 * 2.0 ** -23
    assert float((got - d).abs().max()) <= e * (2 * 1.7149 * 2.92 * 1.5 + 3 * 5.09 * 1.5 + 3) + 2.0 ** -24 * float(d.abs().max())


@pytest.mark.parametrize("batch,cols,rows", [(3, 128, 128), (1, 128, 4000), (2, 300, 260), (1, 1500, 1333), (300, 50, 60), (2, 128, 250), (1, 64, 1000),
                                             (1, 1000, 64), (1, 385, 256), (2, 520, 513), (1, 3000, 128), (9, 515, 1030), (2, 2111, 1700)])
def test_half_intermediates(bl, batch, cols, rows):
    """One float16 matrix each, and sums that stay in tensor memory for as long as they are."""
    g = update_like(batch, cols, rows, cols + rows, "bf16")
    y = bl.newton_schulz(g.cuda(), half_intermediates=True)
    check(y, g, "bf16", store=HALF, additions=max(cols, rows) // 16 + 1)
    assert not torch.equal(y, bl.newton_schulz(g.cuda()))
    space = torch.empty(bl.newton_schulz_workspace_bytes(g, half_intermediates=True), dtype=torch.uint8, device="cuda")
    assert torch.equal(y, bl.newton_schulz(g.cuda(), half_intermediates=True, workspace=space))
    padded = torch.full((batch, cols, rows + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    view = padded[:, :, 1:rows + 1]
    view.copy_(g)
    bl.newton_schulz(view, view, half_intermediates=True)
    assert torch.equal(view, y)
    view.fill_(7.0)
    assert bool((padded == 7.0).all())


def test_half_intermediates_are_for_bfloat16_alone(bl):
    for kind in ("f32", "f16"):
        with pytest.raises(bl.BlasError):
            bl.newton_schulz(torch.ones(4, 4, dtype=TYPES[kind], device="cuda"), half_intermediates=True)
