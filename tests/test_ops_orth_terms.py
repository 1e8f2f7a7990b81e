"""The low halves of the Newton-Schulz pairs (nesle_b200.ops.orthogonalize).

Matrices are kept as two fp16 terms and a product is three tensor-core products,
high by high and both of high by low.  The result's rounding to bf16 hides most of
what a missing term costs, so the tolerance here is close to that rounding.

An output differs from 64 bits by two errors.  The rounding of the result: |r|, its
Frobenius norm, is that of rounding the 64-bit result itself but for the chance of
the entries' low bits, which at 50,000 entries and more moves a norm by less than
1%; 5% are allowed.  And what came before, at most e by the bound of a product kept
in 22 bits (u = 2^-20, 50 u |X|_F a step, times 3.4445 with each later step).  The low
bits know nothing of that error, so squares add: sqrt((1.05 |r|)^2 + e^2)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

A, B, C = 3.4445, -4.7750, 2.0315
STEPS, SCALE = 5, 4096.0


def momentum(rows, cols, device):
    """One direction (of a gradient of rank one) over a floor a thousand times weaker.  What lies beside the weak directions
    grows with them, 485-fold, while the result stays small, and its rounding."""
    g = torch.Generator().manual_seed(rows + cols)
    u, v = torch.randn(rows, generator=g), torch.randn(cols, generator=g)
    return (torch.outer(u / u.norm(), v / v.norm()) + 1e-6 * torch.randn((rows, cols), generator=g)).to(device)


def exact(x):
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.mT if tall else x
    bound = 0.0
    for _ in range(STEPS):
        bound = A * bound + 50 * 2.0 ** -20 * float(torch.linalg.matrix_norm(x))
        g = x @ x.mT
        x = A * x + (B * g + C * (g @ g)) @ x
    x = x.mT if tall else x
    rounding = float(torch.linalg.matrix_norm(x.to(torch.bfloat16).double() - x))
    return x, ((1.05 * rounding) ** 2 + bound ** 2) ** 0.5


def by_terms(x, terms):
    """The operator in 64-bit arithmetic on matrices kept as fp16 pairs; ``terms`` are the products of parts that are taken."""
    def keep(x):
        high = (x * SCALE).half()
        return high.double() / SCALE, (x * SCALE - high.double()).half().double() / SCALE

    def product(a, b):
        return sum(a[i] @ b[j] for i, j in terms)

    def turned(a):
        return a[0].mT, a[1].mT

    x = x.double()
    x = x / (torch.linalg.matrix_norm(x) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    pair = keep(x.mT if tall else x)
    for _ in range(STEPS):
        gram = keep(product(pair, turned(pair)))
        poly = keep(A * torch.eye(gram[0].shape[0], dtype=torch.float64) + B * sum(gram) + C * product(gram, turned(gram)))
        x = product(poly, pair)
        pair = keep(x)
    return (x.mT if tall else x).to(torch.bfloat16).double()


@pytest.mark.parametrize("rows,cols", [(200, 1000), (512, 256), (333, 1500)])
def test_the_tolerance_tells_two_terms_from_one(rows, cols):
    """Restated on the CPU: all three products pass.  Without either low half, or without that of X in P X, they do not; the
    low half of P alone costs less than the result's rounding."""
    x = momentum(rows, cols, "cpu")
    want, tolerance = exact(x)

    def off(terms):
        return float(torch.linalg.matrix_norm(by_terms(x, terms) - want))

    assert off([(0, 0), (0, 1), (1, 0)]) <= tolerance
    for mistaken in ([(0, 0)], [(0, 0), (1, 0)], [(0, 1), (1, 0)]):
        assert off(mistaken) > 2 * tolerance, mistaken


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(200, 1000), (512, 256), (256, 512), (512, 2048), (2048, 512), (333, 1500), (1100, 6500), (3700, 3600)])
def test_products_carry_both_terms(rows, cols):
    """Tiles of 64 columns with and without a cluster, of 128, and of 256 x 256."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nesle_b200 import build, ops

    build.build()
    x = momentum(rows, cols, "cuda")
    want, tolerance = exact(x)
    assert float(torch.linalg.matrix_norm(ops.orthogonalize(x).double() - want)) <= tolerance
