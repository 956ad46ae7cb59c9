"""ops.orthogonalise over its whole range: norms, eps and coefficients far from the usual ones, classes of sizes that the
other tests do not reach, and refusals."""
import pytest
import torch

from mdmm import models, native, ops, ortho
from mdmm.harness import FlatMuon, GradBucket
from test_ortho_gpu import U, check

gpu = pytest.mark.gpu


def test_gradients_are_refused():
    """A matrix that wants a gradient, either way, would lose it."""
    w = torch.ones(4, 4, requires_grad=True)
    with pytest.raises(ValueError, match='gradient'):
        ops.orthogonalise([torch.zeros(4, 4), w])
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match='gradient'):
        ops.orthogonalise([torch.autograd.forward_ad.make_dual(torch.zeros(4, 4), torch.ones(4, 4))])
    for call in (lambda: ops.orthogonalise([w.detach()]), torch.no_grad()(lambda: ops.orthogonalise([w]))):
        with pytest.raises(native.MdmmError):          # (the device's refusal, which comes last)
            call()


def check_scaled(m, got, steps, eps, coefficients=ortho.COEFFICIENTS):
    """check()'s second bound with any eps and coefficients: no more than 8 times the error of the same products in fp32 by
    torch, or than 8 times what one rounding of each iterate's elements costs, and the stored result's own rounding."""
    a, b, c = coefficients

    def iterate(dtype):
        x = m.cpu().to(dtype)
        tall = x.shape[0] > x.shape[1]
        x = x.t() if tall else x
        norm = float(m.double().norm())            # (in 64 bits on both sides: fp32's sum of squares has no range for it)
        x = (x.double() / (norm + eps)).to(dtype)
        kept, flat = [x.double().norm()], [None]
        for _ in range(steps):
            g = x @ x.t()
            p = b * g + c * (g @ g)
            flat.append(float(abs(a) * x.double().norm() + p.double().norm() * x.double().norm()))
            x = a * x + p @ x
            kept.append(float(x.double().norm()))
        return (x.t() if tall else x), flat
    want, flat = iterate(torch.float64)
    plain = iterate(torch.float32)[0].double()
    slope = max(abs(a), 1.0)
    floor = sum(slope ** (steps - k) * U * n for k, n in enumerate(flat) if k)
    near = 8 * max(float((plain - want).norm()), floor) + 64 * U * float(want.norm())
    err = float((got.cpu().double() - want).norm())
    assert err <= near, (err / float(want.norm()), near / float(want.norm()))


@gpu
@pytest.mark.parametrize('norm', [1e-9, 1e-11, 1e-12, 1e-14, 1e-18])
@pytest.mark.parametrize('shape', [(256, 256), (300, 140), (256, 4096), (30, 40)])
def test_norms_far_below_eps(shape, norm):
    """|M| / (|M| + eps) down to 1e-11: the result is as accurate relative to its own size as at any other norm."""
    gen = torch.Generator().manual_seed(21)
    m = torch.randn(shape, generator=gen)
    m = (m * (norm / float(m.double().norm()))).cuda()
    for steps in (0, 1, 5, 9):
        check_scaled(m, ops.orthogonalise([m], steps=steps)[0], steps, 1e-7)


@gpu
@pytest.mark.parametrize('eps,norm', [(0.0, 1e-36), (0.0, 1e37), (1e3, 1e-6), (1e10, 1.0), (1e-30, 1e-34), (1e-7, 1e30)])
def test_any_eps_and_norm(eps, norm):
    gen = torch.Generator().manual_seed(22)
    for shape in ((200, 150), (20, 50), (1100, 1500)):
        m = torch.randn(shape, generator=gen)
        m = (m * (norm / float(m.double().norm()))).cuda()
        n = 2 if shape[0] > 1000 else 1                # (two of them: enough large tiles)
        for o in ops.orthogonalise([m] * n, eps=eps):
            check_scaled(m, o, 5, eps)


@gpu
@pytest.mark.parametrize('coefficients,steps', [((0.0, 1.0, 0.0), 2), ((0.5, 0.0, 0.0), 30), ((0.0, -20.0, 10.0), 1), ((1.5, -0.5, 0.0), 12)])
def test_small_norms_under_other_coefficients(coefficients, steps):
    """Iterations without a linear term, shrinking ones and slow ones, from norms of 1 and far below."""
    gen = torch.Generator().manual_seed(23)
    for norm in (1.0, 1e-9):
        m = torch.randn(170, 140, generator=gen)
        m = (m * (norm / float(m.double().norm()))).cuda()
        check_scaled(m, ops.orthogonalise([m], steps=steps, coefficients=coefficients)[0], steps, 1e-7, coefficients)


@gpu
def test_matrices_of_different_norms_in_one_call():
    gen = torch.Generator().manual_seed(24)
    mats = [(torch.randn(s, generator=gen) * k).cuda() for s, k in (((150, 200), 1.0), ((200, 150), 1e-14), ((20, 30), 1e-13),
                                                                   ((140, 2100), 1e-15), ((150, 200), 1e-3))]
    for m, o in zip(mats, ops.orthogonalise(mats)):
        check_scaled(m, o, 5, 1e-7)


@gpu
def test_muon_leaves_sides_past_the_limit_to_adam():
    """65537 rows: refused as a matrix, Adam's by default (which updates it), before any step."""
    long = torch.nn.Parameter(torch.zeros(65537, 2, device='cuda'))
    short = torch.nn.Parameter(torch.zeros(65536, 2, device='cuda'))
    bucket = GradBucket([short, long])
    with pytest.raises(ValueError, match='65536'):
        FlatMuon(bucket, matrices=[short, long])
    opt = FlatMuon(bucket, adam_lr=0.5)
    assert [g['params'] for g in opt.param_groups] == [[short], [long]]
    bucket.flat.fill_(1.0)
    opt.step()
    assert torch.allclose(long.detach(), torch.full_like(long, -0.5)) and float(short.detach().abs().min()) > 0


def test_the_library_says_why_it_refuses_a_matrix():
    a = native.Ortho()
    a.n = 1
    a.item[0].rows, a.item[0].cols, a.item[0].src_ld, a.item[0].dst_ld = 70000, 5, 5, 5
    codes = [native.lib().mdmm_ortho_ws(a)]
    a.item[0].rows = 0
    codes.append(native.lib().mdmm_ortho_ws(a))
    a.item[0].rows = 7
    assert codes == [-2, -1] and native.lib().mdmm_ortho_ws(a) > 0


@gpu
@pytest.mark.parametrize('cell', ['gru', 'linear'])
def test_muon_leaves_initial_states_to_adam(cell):
    """The default choice on a model with two-layer RNNs: its initial states (2, 1, H) are no matrices."""
    m = models.MultiDKS(['a', 'b'], [3, 4], h_dim=12, z_dim=6, rnn_layers=2, device=torch.device('cuda:0'), rnn_cell=cell)
    opt = FlatMuon(GradBucket(m.parameters()))
    chosen = {id(p) for p in opt.param_groups[0]['params']}
    named = {k: id(p) in chosen for k, p in m.named_parameters()}
    assert all(not named['h0.' + k] for k in 'ab') and {named[k] for k in named if k.endswith('weight')} == {True}


def two_params(cols=3):
    return GradBucket([torch.nn.Parameter(torch.ones(s, device='cuda')) for s in ((5, cols), (7,))])


@gpu
def test_muon_loads_all_of_a_state_or_nothing():
    """A momentum of another shape (one that would broadcast) is refused, and nothing of that state is taken."""
    a, b = two_params(3), two_params(1)
    one, other = FlatMuon(a, matrices=[a.params[0]], lr=0.5), FlatMuon(b, matrices=[b.params[0]], lr=0.25)
    for opt, bucket in ((one, a), (other, b)):
        bucket.flat.fill_(2.0)
        opt.step()
    before = one.state_dict()
    with pytest.raises(ValueError, match='shape'):
        one.load_state_dict(other.state_dict())
    after = one.state_dict()
    assert after['param_groups'] == before['param_groups']
    for i, st in before['state'].items():
        for k, v in st.items():
            assert torch.equal(v, after['state'][i][k])


@gpu
def test_muon_learning_rate_tensors():
    """A loaded learning rate goes into the tensor that a captured step reads; another tensor in its place is noticed before a
    replay."""
    lr, bucket = torch.tensor([0.02], device='cuda'), two_params()
    opt = FlatMuon(bucket, lr=lr, adam_lr=0.5)
    bucket.flat.fill_(1.0)
    opt.step()
    sd = opt.state_dict()
    sd['param_groups'][0] = dict(sd['param_groups'][0], lr=torch.tensor([0.125]))
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        opt.step()
    opt.check_replay()
    opt.load_state_dict(sd)
    assert opt.param_groups[0]['lr'] is lr and float(lr) == 0.125
    opt.check_replay()
    for group, new in ((0, torch.tensor([0.02], device='cuda')), (0, 0.02), (1, torch.tensor([0.5], device='cuda')), (1, 0.25)):
        old, opt.param_groups[group]['lr'] = opt.param_groups[group]['lr'], new
        with pytest.raises(RuntimeError):
            opt.check_replay()
        opt.param_groups[group]['lr'] = old
    opt.check_replay()


@gpu
def test_large_class_with_slices():
    """A matrix whose P X takes large tiles and whose A is summed in slices."""
    gen = torch.Generator().manual_seed(13)
    m = (0.01 * torch.randn(512, 8192, generator=gen)).cuda()
    check(m, ops.orthogonalise([m])[0])
    check(m.t(), ops.orthogonalise([m.t().contiguous()])[0])


@gpu
def test_odd_sizes_on_large_tiles():
    """Both orientations in the large class, beside matrices that its padding or their size keep out of it."""
    gen = torch.Generator().manual_seed(14)
    mats = [(0.01 * torch.randn(s, generator=gen)).cuda() for s in ((1100, 1500), (20, 30), (1500, 1101), (900, 2001), (1099, 1497),
                                                                   (1500, 1100))]
    for m, o in zip(mats, ops.orthogonalise(mats)):
        check(m, o)
