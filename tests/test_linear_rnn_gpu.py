"""MultiDKS with inference RNNs of gated linear recurrences (rnn_cell='linear'), the module they are made of, and FlatMuon,
which trains their matrices."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from mdmm import models, ops, ortho
from mdmm.harness import FlatAdam, FlatMuon, GradBucket, elbo_step
from mdmm.models import common
from mdmm.models.dgts import MultiDGTS

gpu = pytest.mark.gpu


def plain_rnn(rnn, x, h0, mask, reverse):
    """GatedLinearRNN.forward from elementary operations, in the parameters' precision."""
    def norm(v, w):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + 1e-6) * w
    res = F.linear(x, rnn.inp.weight, rnn.inp.bias)
    H = res.shape[-1]
    n = norm(res, rnn.norms[0])
    for k, layer in enumerate(rnn.proj):
        p = F.linear(n, layer.weight, layer.bias)
        f, c, g = p[..., :H], p[..., H:2 * H], p[..., 2 * H:]
        h, hs = h0[k].expand(x.shape[1], H), [None] * len(x)
        for t in (reversed(range(len(x))) if reverse else range(len(x))):
            new = torch.sigmoid(f[t]) * h + torch.sigmoid(-f[t]) * c[t]
            h = new if mask is None else torch.where(mask[t].unsqueeze(-1), new, h)
            hs[t] = h
        res = res + rnn.scales[k] * F.silu(g) * norm(torch.stack(hs), rnn.posts[k])
        if k + 1 < rnn.num_layers:
            n = norm(res, rnn.norms[k + 1])
    return res


@gpu
@pytest.mark.parametrize('layers,bias,masked,reverse', [(1, True, True, True), (2, True, True, False), (3, False, False, True)])
@pytest.mark.parametrize('dims', [(6, 10), (20, 256), (33, 37)])
def test_module_and_gradients(dims, layers, bias, masked, reverse):
    """fp32 operands against 64 bits: a chain of about ten fp32 operations per layer on values of order one, sums of up to 256
    products: 1e-4 of the largest value leaves a factor of ten over u sqrt(256) x 30 operations x 3 layers = 1e-5."""
    torch.manual_seed(sum(dims) + layers)
    T, B = 12, 5
    rnn = common.GatedLinearRNN(dims[0], dims[1], layers, bias).cuda()
    x, h0 = torch.randn(T, B, dims[0]).cuda(), torch.randn(layers, dims[1]).cuda()
    mask = (torch.rand(T, B) > 0.3).cuda() if masked else None
    g = torch.randn(T, B, dims[1]).cuda()
    ref = common.GatedLinearRNN(dims[0], dims[1], layers, bias).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in rnn.state_dict().items()})
    xr, hr = x.double().cpu().requires_grad_(True), h0.double().cpu().requires_grad_(True)
    want = plain_rnn(ref, xr, hr, None if mask is None else mask.cpu(), reverse)
    (want * g.cpu().double()).sum().backward()
    xd, hd = x.requires_grad_(True), h0.requires_grad_(True)
    got = rnn(xd, hd, mask, reverse)
    got.backward(g)
    pairs = [(got, want), (xd.grad, xr.grad), (hd.grad, hr.grad)]
    pairs += [(p.grad, dict(ref.named_parameters())[k].grad) for k, p in rnn.named_parameters()]
    for a, b in pairs:
        b = b.detach()
        assert (a.detach().cpu().double() - b).abs().max() <= 1e-4 * b.abs().max() + 1e-6


@gpu
def test_steps_are_the_module():
    torch.manual_seed(1)
    T, B, D, H, L = 9, 3, 7, 20, 2
    rnn = common.GatedLinearRNN(D, H, L).cuda()
    x, mask = torch.randn(T, B, D).cuda(), (torch.rand(T, B) > 0.3).cuda()
    h0 = torch.randn(L, H).cuda()
    with torch.no_grad():
        want = rnn(x, h0, mask)
    states = h0.unsqueeze(1).repeat(1, B, 1)
    for t in range(T):
        got = rnn.step(x[t], states, mask[t])
        assert (got - want[t]).abs().max() <= 1e-5 * want.abs().max()


@gpu
def test_bf16_operands():
    """The same module with bf16 operands and a bf16 branch: three roundings of 2^-8 a layer on each element, averaged over
    sums of 256: within 3 x 2^-8 x 2 layers = 2.4e-2 of the norm."""
    torch.manual_seed(2)
    T, B, H = 40, 32, 256
    rnn = common.GatedLinearRNN(H, H, 2).cuda()
    x, h0, g = torch.randn(T, B, H).cuda(), torch.zeros(2, H).cuda(), torch.randn(T, B, H).cuda()
    outs = []
    for prec in (None, torch.bfloat16):
        xd = x.clone().requires_grad_(True)
        y = rnn(xd, h0, None, True, prec)
        gs = torch.autograd.grad(y, [xd] + [p for p in rnn.parameters()], g)
        outs.append([y.detach()] + list(gs))
    for a, b in zip(*outs):
        assert float((a - b).norm()) <= 2.4e-2 * float(a.norm()) + 1e-6


def dks(layers, skip, direction, dev, dims=(3, 4)):
    torch.manual_seed(3)
    return models.MultiDKS(['a', 'b'], list(dims), h_dim=12, z_dim=6, rnn_layers=layers, rnn_skip=skip, rnn_dir=direction,
                           device=dev, rnn_cell='linear')


def batch(T=9, lengths=(9, 6, 4), dims=(3, 4)):
    g = torch.Generator().manual_seed(5)
    x = {m: torch.randn(T, len(lengths), d, generator=g) for m, d in zip('ab', dims)}
    for m in x:
        for b, n in enumerate(lengths):
            x[m][n:, b] = float('nan')
    x['a'][2:5, 0] = float('nan')
    mask = torch.arange(T).unsqueeze(1) < torch.tensor(lengths)
    return {k: v.cuda() for k, v in x.items()}, mask.unsqueeze(-1).cuda(), list(lengths)


@gpu
@pytest.mark.parametrize('layers,skip,direction', [(1, True, 'bwd'), (2, True, 'fwd'), (2, False, 'bwd')])
def test_fused_step_is_one_forward_per_pass(layers, skip, direction):
    """MultiDKS.step (shared encoders and RNNs, one combiner launch) against the base class's step of one forward a pass."""
    dev = torch.device('cuda:0')
    m = dks(layers, skip, direction, dev)
    x, mask, lengths = batch()
    found = []
    for step in (m.step, lambda *a, **k: MultiDGTS.step(m, *a, **k)):
        m.zero_grad()
        loss = step(x, mask, 0.7, {'a': 1.0, 'b': 0.5}, lengths=lengths, sample=False)
        loss.backward()
        found.append((float(loss), {k: p.grad.clone() for k, p in m.named_parameters()}))
    assert abs(found[0][0] - found[1][0]) <= 1e-5 * abs(found[1][0])
    for k in found[0][1]:
        a, b = found[0][1][k], found[1][1][k]
        assert (a - b).abs().max() <= 1e-4 * b.abs().max() + 1e-6, k


@gpu
def test_states_reach_only_observed_steps():
    """With skip updates a missing step changes nothing for the others: its content may be anything."""
    dev = torch.device('cuda:0')
    m = dks(1, True, 'bwd', dev)
    feat = torch.randn(6, 2, 12, device=dev)
    mask = torch.ones(6, 2, dtype=torch.bool, device=dev)
    mask[3, 0] = False
    other = feat.clone()
    other[3, 0] = 7.0
    with torch.no_grad():
        a, b = m._rnn('a', feat, mask), m._rnn('a', other, mask)
    keep = torch.ones(6, 2, dtype=torch.bool)
    keep[3, 0] = False
    assert torch.equal(a[keep.cuda()], b[keep.cuda()])


def test_cell_is_checked():
    with pytest.raises(ValueError):
        models.MultiDKS(['a'], [1], rnn_cell='lstm', device=torch.device('cpu'))
    m = models.MultiDKS(['a'], [1], rnn_cell='linear', device=torch.device('cpu'))
    assert isinstance(m.rnn['a'], common.GatedLinearRNN) and m.h0['a'].shape == (1, 1, 32)
    assert isinstance(models.MultiDKS(['a'], [1], device=torch.device('cpu')).rnn['a'], nn.GRU)


# ---- FlatMuon ----------------------------------------------------------------------------------------------------

def plain_muon(params, grads, state, lr, momentum, nesterov, steps, wd, matrices, adam_lr, betas, eps, count):
    for i, (p, g) in enumerate(zip(params, grads)):
        st = state.setdefault(i, {})
        if i in matrices:
            st['m'] = momentum * st.get('m', torch.zeros_like(p)) + g
            u = (g + momentum * st['m'] if nesterov else st['m']).reshape(p.shape[0], -1)
            x = u.t() if u.shape[0] > u.shape[1] else u
            x = x / (x.norm() + 1e-7)
            a, b, c = ortho.COEFFICIENTS
            for _ in range(steps):
                q = x @ x.t()
                x = a * x + (b * q + c * (q @ q)) @ x
            o = x.t() if u.shape[0] > u.shape[1] else x
            p.mul_(1 - lr * wd).sub_(lr * max(1.0, u.shape[0] / u.shape[1]) ** 0.5 * o.reshape(p.shape))
        else:
            st['a'] = betas[0] * st.get('a', torch.zeros_like(p)) + (1 - betas[0]) * g
            st['v'] = betas[1] * st.get('v', torch.zeros_like(p)) + (1 - betas[1]) * g * g
            p.sub_(adam_lr / (1 - betas[0] ** count) * st['a'] / ((st['v'] / (1 - betas[1] ** count)).sqrt() + eps))


SHAPES = [(20, 30), (30,), (40, 10), (8, 3, 4, 4), (1, 9), (5, 5), (300, 70)]


def make_params(dev='cuda'):
    g = torch.Generator().manual_seed(7)
    return [nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dev)) for s in SHAPES]


def fill(params, bucket, k):
    g = torch.Generator().manual_seed(100 + k)
    grads = [torch.randn(p.shape, generator=g) for p in params]
    for p, v in zip(params, grads):
        p.grad = v.to(p.device)
    bucket.check_views()
    return grads


@gpu
@pytest.mark.parametrize('nesterov,wd', [(True, 0.0), (False, 0.1)])
def test_muon_follows_the_formula(nesterov, wd):
    """Six steps against 64 bits.  An update is lr times an orthogonalised matrix whose elements are off by at most 1e-4
    (tests of ops.orthogonalise), so six steps of 0.02 leave 1.2e-5; Adam's side 2e-6 (as FlatAdam's test)."""
    params = make_params()
    bucket = GradBucket(params)
    opt = FlatMuon(bucket, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=wd, adam_lr=1e-2)
    ref = [p.detach().double().cpu() for p in params]
    matrices = [i for i, s in enumerate(SHAPES) if len(s) > 1 and min(s[0], int(torch.tensor(s[1:]).prod())) > 1]
    state = {}
    for k in range(6):
        grads = fill(params, bucket, k)
        opt.step()
        plain_muon(ref, [g.double() for g in grads], state, 0.02, 0.9, nesterov, 5, wd, matrices, 1e-2, (0.9, 0.999), 1e-8, k + 1)
    for p, r in zip(params, ref):
        assert (p.detach().cpu().double() - r).abs().max() < 2e-5


@gpu
@pytest.mark.parametrize('nesterov', [True, False])
def test_muon_of_large_matrices(nesterov):
    """Two steps on matrices that fill the chip with large tiles, beside small ones: as above, with gains up to
    sqrt(4090 / 1000) = 2.1 two steps of 0.02 leave 8.4e-6 and the parameters' rounding."""
    shapes = [(1000, 4096), (4090, 1000), (33, 20), (7,)]
    g = torch.Generator().manual_seed(8)
    params = [nn.Parameter((torch.randn(s, generator=g) * 0.1).cuda()) for s in shapes]
    bucket = GradBucket(params)
    opt = FlatMuon(bucket, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adam_lr=1e-2)
    ref, state = [p.detach().double() for p in params], {}
    for k in range(2):
        grads = fill(params, bucket, k)
        opt.step()
        plain_muon(ref, [v.double().cuda() for v in grads], state, 0.02, 0.9, nesterov, 5, 0.1, [0, 1, 2], 1e-2, (0.9, 0.999), 1e-8,
                   k + 1)
    for p, r in zip(params, ref):
        assert (p.detach().double() - r).abs().max() < 1e-5


@gpu
def test_muon_state_round_trip_and_rest():
    params, others = make_params(), make_params()
    bucket, bo = GradBucket(params), GradBucket(others)
    opt = FlatMuon(bucket, matrices=[params[0], params[6]])
    assert len(opt.param_groups) == 2 and [len(g['params']) for g in opt.param_groups] == [2, 5]
    fill(params, bucket, 0)
    opt.step()
    sd = opt.state_dict()
    back = FlatMuon(bo, matrices=[others[0], others[6]])
    with torch.no_grad():
        for a, b in zip(params, others):
            b.copy_(a)
    back.load_state_dict(sd)
    for b, ps, o in ((bucket, params, opt), (bo, others, back)):
        fill(ps, b, 1)
        o.step()
    for a, b in zip(params, others):
        assert torch.equal(a, b)
    # the parameters that are not its matrices: exactly what FlatAdam makes of them
    solo = make_params()
    bs = GradBucket(solo)
    adam = FlatAdam(bs, lr=1e-3)
    for k in range(2):
        fill(solo, bs, k)
        adam.step()
    for i in (1, 2, 3, 4, 5):
        assert torch.equal(params[i], solo[i])


@gpu
def test_muon_replays_with_a_tensor_learning_rate():
    params, eager = make_params(), make_params()
    bucket, be = GradBucket(params), GradBucket(eager)
    lr = torch.tensor([0.02], device='cuda')
    opt, oe = FlatMuon(bucket, lr=lr), FlatMuon(be, lr=0.02)
    fill(params, bucket, 0)
    fill(eager, be, 0)
    opt.step()
    oe.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 4):
        new = 0.02 / k
        lr.fill_(new)
        oe.param_groups[0]['lr'] = float(lr)
        for b, ps in ((bucket, params), (be, eager)):
            g = torch.Generator().manual_seed(k)
            b.flat.copy_(torch.randn(b.flat.shape, generator=g))
        graph.replay()
        oe.step()
        torch.cuda.synchronize()
        for a, b in zip(params, eager):
            assert torch.equal(a, b)


@gpu
def test_muon_refusals():
    params = make_params()
    bucket = GradBucket(params)
    for kw in ({'momentum': 1.0}, {'ns_steps': -1}, {'matrices': [params[1]]}, {'matrices': [nn.Parameter(torch.ones(3, 3).cuda())]}):
        with pytest.raises(ValueError):
            FlatMuon(bucket, **kw)
    opt = FlatMuon(bucket)
    with pytest.raises(ValueError):
        opt.add_param_group({'params': [nn.Parameter(torch.ones(2, 2).cuda())]})
    params[0].grad = torch.zeros_like(params[0])
    with pytest.raises(RuntimeError):
        opt.step()


def test_muon_needs_the_gpu():
    with pytest.raises(RuntimeError):
        FlatMuon(GradBucket(make_params('cpu')))


@gpu
def test_training_steps_with_muon():
    """A MultiDKS of linear recurrences trained by harness.elbo_step and FlatMuon: the update each step applies is the one
    of the formula for the gradient that it was given."""
    dev = torch.device('cuda:0')
    m = dks(2, True, 'bwd', dev)
    bucket = GradBucket(m.parameters())
    mats = [p for k, p in m.named_parameters() if p.dim() == 2 and k.startswith('rnn.') and 'proj' in k]
    assert len(mats) == 4
    opt = FlatMuon(bucket, lr=0.05, matrices=mats)
    x, mask, lengths = batch()
    before = [p.detach().clone() for p in mats]
    losses = [float(elbo_step(m, opt, bucket, x, mask, lengths, 1.0, {'a': 1.0, 'b': 1.0}, sample=False)) for _ in range(3)]
    assert all(torch.isfinite(torch.tensor(losses)))
    for p, b in zip(mats, before):
        moved = (p.detach() - b).double().cpu()
        # three updates of lr sqrt(3) times a matrix of spectral norm at most 1.3
        assert 0 < float(torch.linalg.matrix_norm(moved, 2)) <= 3 * 0.05 * 3 ** 0.5 * 1.3


@gpu
def test_replayed_training_step():
    """The whole step (model, backward, FlatMuon) replayed from graphs against the eager one."""
    from mdmm.harness import GraphedElboStep
    dev = torch.device('cuda:0')
    x, mask, lengths = batch()
    rec = {'a': 1.0, 'b': 1.0}
    ends = []
    for graphed in (False, True):
        m = dks(2, True, 'bwd', dev)
        bucket = GradBucket(m.parameters())
        opt = FlatMuon(bucket, lr=0.02, matrices=[p for k, p in m.named_parameters() if 'proj' in k and p.dim() == 2])
        if graphed:
            step = GraphedElboStep(m, opt, bucket, x, mask, lengths, 1.0, rec, warmup=2, sample=False)
            losses = [float(step()) for _ in range(3)]
            torch.cuda.synchronize()
        else:
            for _ in range(5):
                last = float(elbo_step(m, opt, bucket, x, mask, lengths, 1.0, rec, sample=False))
        ends.append({k: p.detach().clone() for k, p in m.named_parameters()})
    assert abs(losses[-1] - last) <= 1e-5 * abs(last)
    # the same launches on the same values, but for the division of the gradient (by a device scalar's reciprocal when
    # replayed): a relative 2^-24 of each gradient, which Adam's first steps (a sign) do not amplify beyond lr 1e-3 x 1e-4
    for k in ends[0]:
        assert (ends[0][k] - ends[1][k]).abs().max() <= 1e-5, k


@gpu
@pytest.mark.parametrize('opt_kind', ['muon', 'adam'])
def test_weights_that_an_optimizer_wrote_are_the_ones_used(opt_kind):
    """The module on its own with bf16 operands at a width whose products keep the weight's bf16 copy: after updates through
    the optimizer's launches, outputs and gradients are bit for bit those of a new module of the same weights."""
    torch.manual_seed(4)
    T, B, H = 16, 32, 256
    rnn = common.GatedLinearRNN(H, H, 2).cuda()
    x, h0, g = torch.randn(T, B, H).cuda(), torch.zeros(2, H).cuda(), torch.randn(T, B, H).cuda()
    bucket = GradBucket(rnn.parameters())
    opt = FlatMuon(bucket, lr=0.05) if opt_kind == 'muon' else FlatAdam(bucket, lr=0.05)

    def run(m):
        xd = x.clone().requires_grad_(True)
        y = m(xd, h0, None, False, torch.bfloat16)
        y.backward(g)
        return y.detach(), xd.grad
    for _ in range(3):
        bucket.release()
        got = run(rnn)
        new = common.GatedLinearRNN(H, H, 2).cuda()
        new.load_state_dict(rnn.state_dict())
        for a, b in zip(got, run(new)):
            assert torch.equal(a, b)
        for p, q in zip(rnn.parameters(), new.parameters()):
            assert torch.equal(p.grad, q.grad)
        bucket.check_views()
        versions = [p._version for p in rnn.parameters()]
        opt.step()
        assert all(p._version > v for p, v in zip(rnn.parameters(), versions))


@gpu
def test_replayed_module_uses_the_present_weights():
    """A forward pass captured after eager ones, replayed after updates of the weights: what the eager module gives."""
    torch.manual_seed(5)
    T, B, H = 16, 32, 256
    rnn = common.GatedLinearRNN(H, H, 1).cuda()
    x, h0 = torch.randn(T, B, H).cuda(), torch.zeros(1, H).cuda()
    bucket = GradBucket(rnn.parameters())
    opt = FlatMuon(bucket, lr=0.05)
    with torch.no_grad():
        rnn(x, h0, None, False, torch.bfloat16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = rnn(x, h0, None, False, torch.bfloat16)
    for k in range(3):
        bucket.flat.normal_()
        opt.step()
        graph.replay()
        new = common.GatedLinearRNN(H, H, 1).cuda()
        new.load_state_dict(rnn.state_dict())
        with torch.no_grad():
            want = new(x, h0, None, False, torch.bfloat16)
        torch.cuda.synchronize()
        assert torch.equal(held, want)


@gpu
def test_eager_backward_behind_a_capture():
    """A backward pass of an eager call after another call of the module was captured and not replayed."""
    torch.manual_seed(7)
    T, B, H = 16, 32, 256
    rnn = common.GatedLinearRNN(H, H, 1).cuda()
    x, h0, g = torch.randn(T, B, H).cuda(), torch.zeros(1, H).cuda(), torch.randn(T, B, H).cuda()
    xd = x.clone().requires_grad_(True)
    want = torch.autograd.grad(rnn(xd, h0, None, False, torch.bfloat16), xd, g)[0]
    y = rnn(xd, h0, None, False, torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        rnn(x, h0, None, False, torch.bfloat16)
    assert torch.equal(torch.autograd.grad(y, xd, g)[0], want)


@gpu
@pytest.mark.parametrize('skip', [True, False])
def test_fused_step_with_bf16_operands(skip):
    """MultiDKS.step at a width whose products take bf16 operands (512 rows), the left-out modality's rows too few for them,
    against one forward per pass, which takes them for both: three roundings of 2^-8 a layer on each element of two layers'
    states, 2.4e-2 of a gradient's norm (test_bf16_operands), and on the loss, an average over them, 1e-3."""
    dev = torch.device('cuda:0')
    torch.manual_seed(6)
    m = models.MultiDKS(['a', 'b'], [3, 4], h_dim=256, z_dim=256, rnn_layers=2, rnn_skip=skip, device=dev, rnn_cell='linear')
    m.sweep_dtype = torch.bfloat16
    x, mask, lengths = batch(T=16, lengths=(16,) * 20 + (9,) * 12)
    found = []
    for step in (m.step, lambda *a, **k: MultiDGTS.step(m, *a, **k)):
        m.zero_grad()
        loss = step(x, mask, 0.7, {'a': 1.0, 'b': 0.5}, lengths=lengths, sample=False)
        loss.backward()
        found.append((float(loss), {k: p.grad.clone() for k, p in m.named_parameters()}))
    assert abs(found[0][0] - found[1][0]) <= 1e-3 * abs(found[1][0])
    for k in found[0][1]:
        a, b = found[0][1][k], found[1][1][k]
        assert float((a - b).norm()) <= 2.4e-2 * float(b.norm()) + 1e-6, k
