"""Orthogonalised updates (ops.orthogonalise) against the iteration in 64 bits.

Bound: a step maps singular values by p(s) = a s + b s^3 + c s^5, whose slope is at most a on [0, 1.3] (3.44 at 0, between
-1.6 and 3.44 up to 1.1, 5.4 in size at 1.3, where none of these inputs stays), so an error of X grows by at most a per
step; a step's own rounding is at most G u |X|_F sqrt(K) with K the longest sum (independent roundings) and G = 2 (|a| +
2 |b| 1.7 + 3 |c| 2.9) = 75 from the three products with |X|_2 <= 1.3.  That bound has every rounding aligned with the
steepest direction; beside it the error may be no more than 8 times that of the same products in fp32 by torch, or than
8 times what rounding each iterate's elements once may cost any evaluation that keeps X in fp32: |dX_k|_F <= u |X_k|_F,
grown by a per remaining step, so sum_k a^(steps - k) u |X_k|_F.  (Torch's own error may lie far under that by luck: for
twelve equal rows, eleven zero singular values, it is 1.3e-6 where that sum is (141 |X_1| + 41 |X_2| + 12 |X_3| + 3.4 |X_4| +
|X_5|) u, with every |X_k|_F between 0.7 and 1.2: 8e-6 to 1.4e-5.)
"""
import math

import pytest
import torch

from mdmm import native, ops, ortho

U = 2.0 ** -24
A, B, C = ortho.COEFFICIENTS
gpu = pytest.mark.gpu


def reference(m, steps, dtype=torch.float64, eps=1e-7):
    x = m.to(dtype).reshape(m.shape[0], -1)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    norms = [float(x.norm())]
    for _ in range(steps):
        g = x @ x.t()
        x = A * x + (B * g + C * (g @ g)) @ x
        norms.append(float(x.norm()))
    return (x.t() if tall else x).reshape(m.shape), norms


def check(m, got, steps=5):
    assert got.shape == m.shape and got.dtype == m.dtype
    want, norms = reference(m.cpu(), steps)
    plain = reference(m.cpu().float(), steps, torch.float32)[0]
    err = got.cpu().double() - want
    half = torch.finfo(m.dtype).eps / 2
    K = max(m.shape[0], m.numel() // m.shape[0])
    bound = sum(A ** (steps - k) * 75 * U * math.sqrt(K) * n for k, n in enumerate(norms)) + half * float(want.norm())
    floor = sum(A ** (steps - k) * U * n for k, n in enumerate(norms) if k)
    near = 8 * max(float((plain.double() - want).norm()), floor) + (half + 64 * U) * float(want.norm())
    assert float(err.norm()) <= min(bound, near), (float(err.norm()), bound, near)


SHAPES = [(1, 1), (1, 9), (9, 1), (10, 256), (64, 64), (65, 63), (32, 512), (96, 100), (100, 96), (128, 300), (256, 256),
          (768, 256), (257, 129), (256, 4096), (700, 513)]


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', SHAPES)
def test_orthogonalise(shape, dtype):
    gen = torch.Generator().manual_seed(sum(shape))
    k = max(1, min(shape) // 8)
    m = torch.randn(shape[0], k, generator=gen) @ torch.randn(k, shape[1], generator=gen) + 0.3 * torch.randn(shape, generator=gen)
    m = (0.01 * m).to(dtype).cuda()
    keep = m.clone()
    check(m, ops.orthogonalise([m])[0])
    assert torch.equal(m, keep)


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_orthogonalise_large(dtype):
    gen = torch.Generator().manual_seed(1)
    m = (0.01 * torch.randn(1100, 1500, generator=gen)).to(dtype).cuda()
    check(m, ops.orthogonalise([m])[0])


@gpu
def test_many_matrices_of_any_kind_at_once():
    """More matrices than one launch holds, both types, strided, column-major, four-dimensional and empty ones."""
    gen = torch.Generator().manual_seed(2)
    mats = [torch.randn(s, generator=gen).cuda() for s in [(20, 30), (30, 20), (3, 7), (16, 3, 4, 4), (0, 5), (5, 0)] * 9]
    mats += [torch.randn(40, 50, generator=gen).cuda()[:, ::2], torch.randn(40, 50, generator=gen).cuda()[3:, 5:31],
             torch.randn(40, 50, generator=gen).cuda().t(), torch.randn(1, 50, generator=gen).cuda().expand(12, 50),
             torch.randn(33, 70, generator=gen).bfloat16().cuda()]
    outs = ops.orthogonalise(mats)
    assert len(outs) == len(mats)
    for m, o in zip(mats, outs):
        if m.numel():
            check(m, o)
        else:
            assert o.shape == m.shape
    again = ops.orthogonalise(mats)
    for a, b in zip(outs, again):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize('steps', [0, 1, 2, 7])
def test_steps(steps):
    gen = torch.Generator().manual_seed(3)
    for shape in ((50, 90), (90, 50)):
        m = torch.randn(shape, generator=gen).cuda()
        check(m, ops.orthogonalise([m], steps=steps)[0], steps)


@gpu
def test_singular_values_come_to_one():
    """Five steps of a well-conditioned matrix: every singular value within the band the polynomial maps [0.03, 1] to."""
    gen = torch.Generator().manual_seed(4)
    q = torch.linalg.qr(torch.randn(60, 60, generator=gen, dtype=torch.float64))[0]
    m = (q * torch.linspace(0.3, 1.0, 60, dtype=torch.float64)) @ q.t()
    s = torch.linspace(0.3, 1.0, 60, dtype=torch.float64)
    s = s / s.norm()
    for _ in range(5):
        s = A * s + B * s ** 3 + C * s ** 5
    got = torch.linalg.svdvals(ops.orthogonalise([m.float().cuda()])[0].cpu().double())
    assert (got.sort().values - s.sort().values).abs().max() < 1e-4        # (the bound above at K = 60: 2e-3 / sqrt(60) each)
    assert 0.6 < float(got.min()) and float(got.max()) < 1.3


@gpu
def test_zero_nan_and_huge():
    """A zero matrix gives zeros; NaN stays in its own matrix; the scale of a matrix does not matter."""
    gen = torch.Generator().manual_seed(5)
    a = torch.randn(30, 40, generator=gen).cuda()
    bad = a.clone()
    bad[3, 4] = float('nan')
    z, b, x, big, small = ops.orthogonalise([torch.zeros_like(a), bad, a, a * 1e12, a * 1e-3])
    assert not z.any() and torch.isnan(b).any()
    check(a, x)
    check(a * 1e12, big)
    check(a * 1e-3, small)


@gpu
def test_replayed_from_a_graph():
    gen = torch.Generator().manual_seed(6)
    mats = [torch.randn(s, generator=gen).cuda() for s in ((70, 100), (200, 30))]
    ops.orthogonalise(mats)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.orthogonalise(mats)
    for _ in range(3):
        for m in mats:
            m.copy_(torch.randn(m.shape, generator=gen))
        want = [t.clone() for t in ops.orthogonalise(mats)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize('call', [
    lambda: ops.orthogonalise([torch.zeros(5)]),
    lambda: ops.orthogonalise([torch.zeros(5, 5).double()]),
    lambda: ops.orthogonalise([torch.zeros(5, 5, dtype=torch.float16)]),
    lambda: ops.orthogonalise([torch.zeros(5, 5)], steps=-1),
    lambda: ops.orthogonalise([torch.zeros(5, 5)], steps=2.5),
    lambda: ops.orthogonalise([torch.zeros(5, 5)], coefficients=(1.0, 2.0)),
    lambda: ops.orthogonalise([torch.zeros(1).expand(70000, 5)]),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_no_cpu_fallback():
    assert ops.orthogonalise([]) == []
    with pytest.raises(native.MdmmError):
        ops.orthogonalise([torch.zeros(4, 4)])


@gpu
@pytest.mark.parametrize('coefficients', [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5)])
def test_other_coefficients(coefficients):
    """Polynomials that map [0, 1] to itself with slopes up to a there: the module's first bound with their own G."""
    a, b, c = coefficients
    gen = torch.Generator().manual_seed(7)
    m = torch.randn(70, 130, generator=gen)
    x = m.double() / (m.double().norm() + 1e-7)
    bound = 0.0
    for k in range(6):
        bound = a * bound + 2 * (a + 2 * abs(b) + 3 * abs(c)) * U * math.sqrt(130) * float(x.norm())
        if k < 5:
            g = x @ x.t()
            x = a * x + (b * g + c * (g @ g)) @ x
    got = ops.orthogonalise([m.cuda()], coefficients=coefficients)[0].cpu().double()
    assert float((got - x).norm()) <= bound


@pytest.mark.parametrize('call', [
    lambda: ops.orthogonalise([torch.zeros(5, 5)], steps=1001),
    lambda: ops.orthogonalise([torch.zeros(5, 5)], coefficients=(float('nan'), 0.0, 0.0)),
    lambda: ops.orthogonalise([torch.zeros(5, 5)], coefficients=(4.0, 0.0, 0.0)),           # 4 after a step
    lambda: ops.orthogonalise([torch.zeros(5, 5)], coefficients=(3.4445, -4.775, 2.6)),     # 1.27, then 3.2
    lambda: ops.orthogonalise([torch.zeros(5, 5)], coefficients=(1.0, 0.0, 16.0)),          # P = 16 in the first step
])
def test_diverging_iterations_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_bounded_iterations_are_not_refused():
    for c in (ortho.COEFFICIENTS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (1.0, 0.0, 0.0), (0.0, 0.0, 0.0)):
        with pytest.raises(native.MdmmError):         # (the device's refusal, which comes last)
            ops.orthogonalise([torch.zeros(4, 4)], coefficients=c)


@gpu
@pytest.mark.parametrize('shape', [(7, 146), (146, 7), (5, 300), (27, 2), (40, 256), (64, 4096), (4096, 33), (64, 65), (65, 64)])
def test_short_sides(shape):
    """Shorter sides about one tile of 64, with the longer side in one piece and in several; the iterate after 0 steps too."""
    gen = torch.Generator().manual_seed(8 + sum(shape))
    m = (0.02 * torch.randn(shape, generator=gen)).cuda()
    keep = m.clone()
    for steps in (0, 1, 5):
        check(m, ops.orthogonalise([m], steps=steps)[0], steps)
    assert torch.equal(m, keep)


@gpu
def test_large_and_small_together():
    """Enough large matrices for the large tile, of odd sizes and both orientations, beside small ones."""
    gen = torch.Generator().manual_seed(12)
    mats = [(0.01 * torch.randn(s, generator=gen)).cuda() for s in ((1100, 1500), (20, 30), (1500, 1101), (900, 2001), (200, 70))]
    for m, o in zip(mats, ops.orthogonalise(mats)):
        check(m, o)
