"""The gated linear recurrence, the block norms and the layer that joins them (mdmm.recurrent) against 64-bit formulas.

Tolerances are running error bounds: with u = 2^-24, a state is a sum of terms that were each multiplied by some a's, and
every step adds at most 8 u of the terms' absolute sum (a and k are formed to 4 u each, one product, one sum, and a share
for the products of a's that a scan over pieces forms), so e_t = a_t e_{t-1} + 8 u S_t with S_t = a_t S_{t-1} + k_t |c_t|;
the adjoint the same way.  A stored tensor adds half a step of its type.
"""
import os
import subprocess
import sys

import pytest
import torch

from mdmm import native, ops

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
gpu = pytest.mark.gpu


def make(gen, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype)


def scan_ref(gates, h0, mask, reverse, g_h=None, g_last=None):
    """64-bit states and gradients with their error bounds: dict name -> (value, bound)."""
    T, B, H2 = gates.shape
    H = H2 // 2
    f, c = gates[..., :H].double(), gates[..., H:].double()
    m = torch.ones(T, B, 1, dtype=torch.bool) if mask is None else (mask != 0).unsqueeze(-1)
    a = torch.where(m, torch.sigmoid(f), torch.ones_like(f))
    k = torch.where(m, torch.sigmoid(-f), torch.zeros_like(f))
    c = torch.where(m, c, torch.zeros_like(c))
    h = torch.zeros(B, H, dtype=torch.float64) if h0 is None else h0.double().expand(B, H).clone()
    s, e = h.abs(), torch.zeros_like(h)
    order = list(range(T))[::-1] if reverse else list(range(T))
    hs, es, before, e_before = (torch.zeros(T, B, H, dtype=torch.float64) for _ in range(4))
    for t in order:
        before[t], e_before[t] = h, e
        h, s = a[t] * h + k[t] * c[t], a[t] * s + k[t] * c[t].abs()
        e = a[t] * e + 8 * U * s
        hs[t], es[t] = h, e
    out = {'h': (hs, es), 'last': (h, e)}
    if g_h is None and g_last is None:
        return out
    zero = torch.zeros(B, H, dtype=torch.float64)
    d = zero if g_last is None else g_last.double()
    s, e = d.abs(), zero
    df, dc, e_df, e_dc = (torch.zeros(T, B, H, dtype=torch.float64) for _ in range(4))
    for t in order[::-1]:
        g = zero if g_h is None else g_h[t].double()
        G, s = g + d, g.abs() + s
        e = e + 8 * U * s
        dc[t], e_dc[t] = G * k[t], e * k[t] + 8 * U * s * k[t]
        diff = before[t] - c[t]
        df[t] = G * diff * a[t] * k[t]
        e_df[t] = a[t] * k[t] * (e * diff.abs() + s * e_before[t] + 16 * U * s * (before[t].abs() + c[t].abs()))
        d, s, e = a[t] * G, a[t] * s, a[t] * e + 4 * U * a[t] * s
    out['gates'] = (torch.cat([df, dc], -1), torch.cat([e_df, e_dc], -1))
    if h0 is not None:
        if h0.dim() == 1:
            out['h0'] = (d.sum(0), e.sum(0) + (B + 8) * U * s.sum(0))
        else:
            out['h0'] = (d, e)
    return out


def close(got, want, name=''):
    value, bound = want
    got64 = got.detach().cpu().double()
    assert got64.shape == value.shape, (name, got64.shape, value.shape)
    tol = bound + HALF[got.dtype] * (value.abs() + bound) + 1e-37
    bad = ~((got64 - value).abs() <= tol)
    assert not bad.any(), '%s: %d of %d off, worst %.3g of its bound' % (
        name, int(bad.sum()), bad.numel(), float(((got64 - value).abs() / tol).nan_to_num(1e30).max()))


def to(dev, t):
    return None if t is None else t.to(dev)


MASKS = ('none', 'ragged', 'holes', 'nothing')


def make_mask(kind, T, B, gen):
    if kind == 'none':
        return None
    if kind == 'nothing':
        return torch.zeros(T, B, dtype=torch.bool)
    if kind == 'ragged':
        n = torch.randint(0, T + 1, (B,), generator=gen)
        return torch.arange(T).unsqueeze(1) < n
    return torch.rand(T, B, generator=gen) > 0.3


SCANS = [(1, 1, 1), (1, 5, 7), (2, 3, 64), (7, 4, 33), (8, 2, 20), (9, 1, 130), (40, 16, 256), (63, 3, 6), (64, 2, 12),
         (65, 3, 5), (129, 2, 66), (300, 1, 3), (1000, 1, 4), (1025, 2, 130), (4100, 1, 8)]


@gpu
@pytest.mark.parametrize('T,B,H', SCANS)
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('mask', MASKS)
def test_scan_and_gradients(T, B, H, dtype, mask):
    for reverse, h0_kind in ((False, 'row'), (True, 'full'), (True, 'none')):
        gen = torch.Generator().manual_seed(T * 7 + B * 3 + H)
        gates = torch.cat([make(gen, T, B, H, std=1.5, mean=2.0), make(gen, T, B, H)], -1).to(dtype)
        m = make_mask(mask, T, B, gen)
        h0 = {'row': make(gen, H), 'full': make(gen, B, H), 'none': None}[h0_kind]
        g_h, g_last = make(gen, T, B, H, dtype=dtype), make(gen, B, H)
        want = scan_ref(gates, h0, m, reverse, g_h, g_last)
        leaves = [to('cuda', gates).requires_grad_(True)]
        if h0 is not None:
            leaves.append(to('cuda', h0).requires_grad_(True))
        h, last = ops.gated_scan(leaves[0], leaves[1] if h0 is not None else None, mask=to('cuda', m), reverse=reverse)
        assert h.dtype == dtype and last.dtype == F32
        grads = torch.autograd.grad([h, last], leaves, [g_h.cuda(), g_last.cuda()])
        close(h, want['h'], 'h')
        close(last, want['last'], 'last')
        close(grads[0], want['gates'], 'gates')
        if h0 is not None:
            close(grads[1], want['h0'], 'h0')


@gpu
def test_scan_takes_nothing_from_masked_steps():
    """NaN and infinities where the mask is 0 change nothing: outputs and gradients bit for bit those of zeros there."""
    gen = torch.Generator().manual_seed(5)
    T, B, H = 70, 3, 10
    gates, m = make(gen, T, B, 2 * H), torch.rand(T, B, generator=gen) > 0.4
    g = make(gen, T, B, H).cuda()
    outs = []
    for fill in (0.0, float('nan'), float('inf'), -float('inf'), torch.finfo(F32).min):
        x = torch.where(m.unsqueeze(-1), gates, torch.full_like(gates, fill)).cuda().requires_grad_(True)
        h, last = ops.gated_scan(x, mask=m.cuda())
        outs.append((h, last, torch.autograd.grad(h, x, g)[0]))
    for o in outs[1:]:
        for a, b in zip(outs[0], o):
            assert torch.equal(a, b)


@gpu
def test_scan_saturated_gates():
    """Infinite and extreme logits: a of exactly 0 and 1, finite states and gradients."""
    f = torch.tensor([-float('inf'), -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, float('inf')]).view(1, 1, -1)
    f, c = f.repeat(6, 2, 1), torch.ones(6, 2, 9) * 0.5
    x = torch.cat([f, c], -1)
    want = scan_ref(x, torch.ones(9), None, False, torch.ones(6, 2, 9))
    xd = x.cuda().requires_grad_(True)
    h, _ = ops.gated_scan(xd, torch.ones(9, device='cuda'))
    close(h, want['h'])
    close(torch.autograd.grad(h, xd, torch.ones(6, 2, 9, device='cuda'))[0], want['gates'])


@gpu
def test_scan_strided_inputs_and_float_mask():
    gen = torch.Generator().manual_seed(6)
    T, B, H = 37, 5, 12
    base = make(gen, B, T, 2 * H + 3)                       # (batch first, columns of a wider row)
    m = (torch.rand(T, B, 1, generator=gen) > 0.3).float()
    x = base.cuda()[..., 1:1 + 2 * H].transpose(0, 1)
    h0 = make(gen, 2 * H, B).cuda()[::2].t()
    want = scan_ref(base[..., 1:1 + 2 * H].transpose(0, 1), h0.cpu(), m.squeeze(-1), True)
    h, last = ops.gated_scan(x, h0, mask=m.cuda(), reverse=True)
    close(h, want['h'])
    close(last, want['last'])
    row = make(gen, 1, B, 2 * H).cuda().expand(T, B, 2 * H).requires_grad_(True)     # one row for every step
    h, _ = ops.gated_scan(row)
    want = scan_ref(row.detach().cpu(), None, None, False, torch.ones(T, B, H))
    close(h, want['h'])
    close(torch.autograd.grad(h.sum(), row)[0], want['gates'])


@gpu
def test_scan_over_sequences_2_gib_apart():
    """Gates whose sequences lie 2 GiB apart (a step's offsets do not fit 31 bits) against a compact copy."""
    gen = torch.Generator().manual_seed(14)
    T, B, H = 70, 3, 6
    far = 2 ** 29
    room = torch.empty((B - 1) * far + T * 2 * H, device='cuda')
    wide = room.as_strided((T, B, 2 * H), (2 * H, far, 1))
    wide.copy_(make(gen, T, B, 2 * H))
    g = make(gen, T, B, H).cuda()
    for reverse in (False, True):
        outs = []
        for x in (wide.detach(), wide.contiguous()):
            x.requires_grad_(True)
            h, last = ops.gated_scan(x, reverse=reverse)
            outs.append((h, last, torch.autograd.grad(h, x, g)[0]))
        for a, b in zip(*outs):
            assert torch.equal(a, b)


@gpu
def test_scan_past_32_bits():
    """4.8e9 gates: the last steps of the whole scan against a scan of them alone from the state in front of them.  The two
    group their steps differently: 1e-5 covers fp32 sums of values of order one, the bf16 outputs a rounding each."""
    T, B, H, k = 9200, 512, 512, 37
    gates = torch.empty(T, B, 2 * H, device='cuda', dtype=BF16)
    for i in range(0, T, 400):
        gates[i:i + 400].normal_()
    assert gates.numel() > 2 ** 32
    with torch.no_grad():
        h, last = ops.gated_scan(gates)
        _, state = ops.gated_scan(gates[:T - k])
        tail, end = ops.gated_scan(gates[T - k:], state)
    assert (last - end).abs().max() <= 1e-5
    assert ((h[T - k:].float() - tail.float()).abs() <= 1e-5 + 2 * HALF[BF16] * tail.float().abs()).all()


@gpu
def test_norm_past_32_bits():
    rows, H = 3600000, 1200
    x = torch.empty(rows, H, device='cuda', dtype=BF16)
    for i in range(0, rows, 200000):
        x[i:i + 200000].normal_()
    assert x.numel() > 2 ** 32
    w = torch.linspace(0.5, 1.5, H, device='cuda')
    with torch.no_grad():
        n = ops.rms_norm(x, w)
        assert torch.equal(n[-1000:], ops.rms_norm(x[-1000:], w)) and torch.equal(n[:1000], ops.rms_norm(x[:1000], w))


@gpu
@pytest.mark.parametrize('shape', [(0, 3, 8), (4, 0, 8), (4, 3, 0)])
def test_scan_empty(shape):
    T, B, H = shape
    x = torch.zeros(T, B, 2 * H, device='cuda', requires_grad=True)
    h0 = torch.randn(H, device='cuda', requires_grad=True)
    h, last = ops.gated_scan(x, h0)
    assert h.shape == (T, B, H) and last.shape == (B, H)
    if T == 0:
        assert torch.equal(last, h0.expand(B, H))
    g = torch.autograd.grad([h, last], [x, h0], [torch.ones_like(h), torch.ones_like(last)])
    assert g[0].shape == x.shape and torch.equal(g[1], torch.full((H,), float(B) if T == 0 else 0.0, device='cuda'))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_scan_steps_are_the_scan(dtype):
    """T single steps, the state updated in place, against one scan over them."""
    gen = torch.Generator().manual_seed(8)
    T, B, H = 11, 6, 40
    x, m = make(gen, T, B, 2 * H, dtype=dtype).cuda(), (torch.rand(T, B, generator=gen) > 0.3).cuda()
    want = scan_ref(x.cpu(), torch.ones(B, H), m.cpu(), False)
    state = torch.ones(B, H, device='cuda')
    for t in range(T):
        h, new = ops.gated_scan_step(x[t], state, mask=m[t], new_state=state)
        assert new is state
        close(h, (want['h'][0][t], want['h'][1][t]))
    close(state, want['last'])
    h, new = ops.gated_scan_step(x[0], torch.ones(B, H, device='cuda'))
    assert new.data_ptr() != state.data_ptr() and h.dtype == dtype


@gpu
def test_scan_gradient_by_differences():
    """The gradient of a weighted sum of the states against central differences, taken in 64 bits."""
    gen = torch.Generator().manual_seed(9)
    T, B, H = 13, 2, 3
    x, h0, w = make(gen, T, B, 2 * H), make(gen, H), make(gen, T, B, H)
    xd, hd = x.cuda().requires_grad_(True), h0.cuda().requires_grad_(True)
    h, _ = ops.gated_scan(xd, hd)
    gx, gh = torch.autograd.grad(h, [xd, hd], w.cuda())

    def loss(x_, h_):
        return float((scan_ref(x_, h_, None, False)['h'][0] * w.double()).sum())
    # the difference quotient's own error: step^2 / 6 times a third derivative (below 10 here) + 2^-52 / step
    step, tol = 1e-4, 1e-6
    for idx in ((0, 0, 0), (5, 1, 2), (12, 0, 4), (7, 1, 5)):
        d = torch.zeros_like(x).double()
        d[idx] = step
        num = (loss(x.double() + d, h0.double()) - loss(x.double() - d, h0.double())) / (2 * step)
        assert abs(float(gx[idx]) - num) < tol + 1e-5 * abs(num)
    d = torch.zeros(H).double()
    d[1] = step
    num = (loss(x.double(), h0.double() + d) - loss(x.double(), h0.double() - d)) / (2 * step)
    assert abs(float(gh[1]) - num) < tol + 1e-5 * abs(num)


# ---- norms -------------------------------------------------------------------------------------------------------

def norm_ref(y, res, w, gate, s, w2, eps, g_out=None, g_n=None):
    """64-bit block norm and gradients by autograd, and magnitudes: the same expressions with every term's absolute value,
    which times 64 u bounds a rounding per operation (about 30 along the longest chain) with first-order growth.
    y None: the plain norm of res."""
    dbl = lambda t: None if t is None else t.double().detach().requires_grad_(True)     # noqa: E731
    y, res, w, gate, s, w2 = (dbl(t) for t in (y, res, w, gate, s, w2))
    H = res.shape[-1]
    r = act = 1.0
    out, m_out = res, res.abs()
    if y is not None:
        r = torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps)
        act = 1.0 if gate is None else gate * torch.sigmoid(gate)
        branch = (1.0 if s is None else s) * act * (y * r * w)
        out, m_out = res + branch, res.abs() + branch.abs()
    val, mag = {'out': out}, {'out': m_out}
    r2 = 0.0
    if w2 is not None:
        r2 = torch.rsqrt(out.pow(2).mean(-1, keepdim=True) + eps)
        grow = 1 + m_out.norm(dim=-1, keepdim=True) / (out.norm(dim=-1, keepdim=True) + 1e-300)
        val['n'], mag['n'] = out * r2 * w2, (m_out + out.abs() * grow) * r2 * w2.abs()
    if g_out is None and g_n is None:
        return val, mag
    go = torch.zeros_like(out) if g_out is None else g_out.double()
    total = (out * go).sum()
    m_d = go.abs()
    red = lambda t: t.reshape(-1, H).sum(0)                                              # noqa: E731
    if g_n is not None:
        total = total + (val['n'] * g_n.double()).sum()
        q = (g_n.double() * w2).abs()
        m_d = m_d + grow * r2 * (q + m_out * r2 * r2 * (q * m_out).mean(-1, keepdim=True))
        mag['w2'] = red((g_n.double().abs() * m_out * r2) * grow)
    mag['res'] = m_d
    if y is not None:
        sc = 1.0 if s is None else s.abs()
        aa = 1.0 if gate is None else act.abs()
        x = (y * r).abs()
        if s is not None:
            mag['s'] = red(m_d * aa * x * w.abs())
        if gate is not None:
            mag['gate'] = m_d * sc * x * w.abs() * (1 + gate.abs())
        t = m_d * sc * aa
        mag['w'] = red(t * x)
        mag['y'] = r * (t * w.abs() + x * (t * w.abs() * x).mean(-1, keepdim=True))
    names = [k for k, v in (('y', y), ('res', res), ('w', w), ('gate', gate), ('s', s), ('w2', w2)) if v is not None
             and not (k == 'w2' and g_n is None)]
    if y is None:
        names = [k for k in names if k in ('res', 'w2')]
    leaves = {'y': y, 'res': res, 'w': w, 'gate': gate, 's': s, 'w2': w2}
    for k, g in zip(names, torch.autograd.grad(total, [leaves[k] for k in names])):
        val[k] = g
    return val, mag


def near(got, val, mag, key, rows=1):
    """rows: the most terms one thread adds up for a column sum (each sum a rounding of at most u of the absolute sum)."""
    close(got, (val[key].detach(), (64 + rows) * U * mag[key].detach()), key)


NORMS = [(1, 1), (1, 256), (5, 7), (3, 64), (17, 333), (130, 256), (9, 512), (33, 1000), (4, 1023), (6, 1028), (5, 2048),
         (3, 2500), (2, 4096), (2, 4100), (2, 5001), (1, 8192), (2500, 20)]
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32)]


@gpu
@pytest.mark.parametrize('rows,H', NORMS)
@pytest.mark.parametrize('dtype,res_dtype', TYPES)
def test_block_norm_and_gradients(rows, H, dtype, res_dtype):
    for has_gate, has_scale, has_next in ((True, True, True), (False, False, False), (True, False, True), (False, True, False)):
        gen = torch.Generator().manual_seed(rows + H)
        y, res = make(gen, rows, H, dtype=dtype), make(gen, rows, H, dtype=res_dtype)
        w = make(gen, H, std=0.1, mean=1.0)
        gate = make(gen, rows, H, dtype=dtype) if has_gate else None
        s = make(gen, H, std=0.1, mean=0.5) if has_scale else None
        w2 = make(gen, H, std=0.1, mean=1.0) if has_next else None
        g_out = make(gen, rows, H, dtype=res_dtype)
        g_n = make(gen, rows, H, dtype=dtype) if has_next else None
        val, mag = norm_ref(y, res, w, gate, s, w2, 1e-6, g_out, g_n)
        ins = {'y': y, 'res': res, 'w': w, 'gate': gate, 's': s, 'w2': w2}
        dev = {k: to('cuda', v) for k, v in ins.items()}
        leaves = {k: v.requires_grad_(True) for k, v in dev.items() if v is not None}
        got = ops.block_norm(dev['y'], dev['res'], dev['w'], gate=dev['gate'], scale=dev['s'], next_weight=dev['w2'])
        outs = got if has_next else (got,)
        near(outs[0], val, mag, 'out')
        if has_next:
            near(outs[1], val, mag, 'n')
        grads = torch.autograd.grad(outs, list(leaves.values()), [g.cuda() for g in (g_out, g_n) if g is not None])
        for k, g in zip(leaves, grads):
            near(g, val, mag, k, rows=rows)


@gpu
@pytest.mark.parametrize('rows,H', [(1, 1), (10, 33), (257, 256), (3, 8192), (64, 1280)])
@pytest.mark.parametrize('dtype,out', [(F32, F32), (BF16, BF16), (F32, BF16)])
def test_rms_norm_and_gradients(rows, H, dtype, out):
    gen = torch.Generator().manual_seed(rows * 5 + H)
    x, w, g = make(gen, rows, H, dtype=dtype), make(gen, H, std=0.1, mean=1.0), make(gen, rows, H, dtype=out)
    val, mag = norm_ref(None, x, None, None, None, w, 1e-6, None, g)
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    n = ops.rms_norm(xd, wd, dtype=out)
    assert n.dtype == out
    near(n, val, mag, 'n')
    gx, gw = torch.autograd.grad(n, [xd, wd], g.cuda())
    near(gx, val, mag, 'res')
    near(gw, val, mag, 'w2', rows=rows)


@gpu
def test_norms_strided_rows_and_partial_gradients():
    """Column slices of wider rows (also ones whose rows are not 16-byte aligned), one row for all, gradients of some
    inputs alone and of one output alone."""
    gen = torch.Generator().manual_seed(11)
    for lo in (0, 4, 3):
        wide = make(gen, 6, 5, 40)
        y, gate = wide[..., lo:lo + 12], wide[..., 20 + lo:32 + lo]
        res, w, w2 = make(gen, 12).expand(6, 5, 12), make(gen, 12), make(gen, 12)
        g_n = make(gen, 6, 5, 12)
        val, mag = norm_ref(y, res, w, gate, None, w2, 1e-6, None, g_n)
        wd = wide.cuda()
        yd, gd = wd[..., lo:lo + 12].requires_grad_(True), wd[..., 20 + lo:32 + lo].requires_grad_(True)
        w2d = w2.cuda().requires_grad_(True)
        out, n = ops.block_norm(yd, res.cuda(), w.cuda(), gate=gd, next_weight=w2d)
        near(out, val, mag, 'out')
        near(n, val, mag, 'n')
        for k, g in zip(('y', 'gate', 'w2'), torch.autograd.grad(n, [yd, gd, w2d], g_n.cuda())):
            near(g, val, mag, k, rows=30)


@gpu
def test_norm_of_zero_and_extreme_rows():
    """A zero row: eps alone under the root, zeros out and finite gradients.  Rows of 1e15 and 1e-15 stay apart (rows are
    independent)."""
    x = torch.zeros(3, 16)
    x[1], x[2] = 1e15, 1e-15
    w = torch.ones(16)
    g = torch.ones(3, 16)
    val, mag = norm_ref(None, x, None, None, None, w, 1e-6, None, g)
    xd = x.cuda().requires_grad_(True)
    n = ops.rms_norm(xd, w.cuda())
    near(n, val, mag, 'n')
    near(torch.autograd.grad(n, xd, g.cuda())[0], val, mag, 'res')


@gpu
def test_norms_without_rows():
    w = torch.ones(8, device='cuda', requires_grad=True)
    y, res = torch.zeros(0, 4, 8, device='cuda', requires_grad=True), torch.zeros(0, 4, 8, device='cuda', requires_grad=True)
    out, n = ops.block_norm(y, res, w, next_weight=w)
    assert out.shape == n.shape == (0, 4, 8)
    gy, gw = torch.autograd.grad([out, n], [y, w], [out, n])
    assert gy.shape == y.shape and torch.equal(gw, torch.zeros_like(w))


# ---- the layer ---------------------------------------------------------------------------------------------------

def layer_ref(proj, res, h0, w, s, w2, mask, reverse, g_out, g_n, g_last):
    H = res.shape[-1]
    scan = scan_ref(proj[..., :2 * H], h0, mask, reverse)
    h, e_h = scan['h']
    val, mag = norm_ref(h, res, w, proj[..., 2 * H:], s, w2, 1e-6, g_out, g_n)
    back = scan_ref(proj[..., :2 * H], h0, mask, reverse, val['y'], g_last)
    return val, mag, scan, back


@gpu
@pytest.mark.parametrize('T,B,H', [(1, 1, 3), (5, 3, 20), (40, 8, 256), (70, 2, 33), (200, 1, 64), (33, 3, 300), (17, 2, 516),
                                   (130, 2, 1030)])
@pytest.mark.parametrize('dtype,res_dtype', TYPES)
@pytest.mark.parametrize('mask', ['none', 'ragged', 'nothing'])
def test_block_is_scan_and_norm(T, B, H, dtype, res_dtype, mask):
    """The layer against the two formulas in a row.  The state's own error (1e-6 of its size at these lengths; a state near
    zero in a whole row would amplify it, random rows are not) enters the norm: a flat 1e-5 of the largest value is allowed
    on top of the types' half steps, where fp32 intermediates leave about 1e-6."""
    gen = torch.Generator().manual_seed(T + B + H)
    reverse = bool(T % 2)
    proj = torch.cat([make(gen, T, B, H, mean=1.0), make(gen, T, B, 2 * H)], -1).to(dtype)
    res, h0 = make(gen, T, B, H, dtype=res_dtype), make(gen, H)
    w, s, w2 = (make(gen, H, std=0.1, mean=1.0) for _ in range(3))
    m = make_mask(mask, T, B, gen)
    g_out, g_n, g_last = make(gen, T, B, H, dtype=res_dtype), make(gen, T, B, H, dtype=dtype), make(gen, B, H)
    val, mag, scan, back = layer_ref(proj, res, h0, w, s, w2, m, reverse, g_out, g_n, g_last)
    d = [t.cuda().requires_grad_(True) for t in (proj, res, h0, w, s, w2)]
    out, n, last = ops.gated_block(d[0], d[1], d[2], d[3], scale=d[4], next_weight=d[5], mask=to('cuda', m), reverse=reverse)
    assert out.dtype == res_dtype and n.dtype == dtype and last.dtype == F32
    grads = torch.autograd.grad([out, n, last], d, [g_out.cuda(), g_n.cuda(), g_last.cuda()])
    d_proj = torch.cat([back['gates'][0], val['gate']], -1)
    for name, got, want in (('out', out, val['out']), ('n', n, val['n']), ('last', last, scan['last'][0]),
                            ('proj', grads[0], d_proj), ('res', grads[1], val['res']), ('h0', grads[2], back['h0'][0]),
                            ('w', grads[3], val['w']), ('s', grads[4], val['s']), ('w2', grads[5], val['w2'])):
        want = want.detach()
        err = (got.detach().cpu().double() - want).abs()
        tol = 1e-5 * want.abs().max() + HALF[got.dtype] * want.abs()
        assert (err <= tol).all(), (name, float(err.max()), float(want.abs().max()))


@gpu
@pytest.mark.parametrize('H', [3, 256, 300, 1100])
@pytest.mark.parametrize('dtype,res_dtype', TYPES)
def test_block_steps_are_the_block(H, dtype, res_dtype):
    gen = torch.Generator().manual_seed(H)
    T, B = 5, 4
    proj, res = make(gen, T, B, 3 * H, dtype=dtype).cuda(), make(gen, T, B, H, dtype=res_dtype).cuda()
    w, s, w2 = (make(gen, H, std=0.1, mean=1.0).cuda() for _ in range(3))
    m = (torch.rand(T, B, generator=gen) > 0.3).cuda()
    with torch.no_grad():
        out, n, last = ops.gated_block(proj, res, torch.ones(B, H, device='cuda'), w, scale=s, next_weight=w2, mask=m)
        state = torch.ones(B, H, device='cuda')
        for t in range(T):
            o, q, state = ops.gated_block_step(proj[t], res[t], state, w, scale=s, next_weight=w2, mask=m[t], new_state=state)
            for got, want in ((o, out[t]), (q, n[t])):
                # the same formula with sums in another order: 1e-5 of the largest value, and a rounding either way
                tol = 1e-5 * want.float().abs().max() + 2 * HALF[got.dtype] * want.float().abs()
                assert ((got.float() - want.float()).abs() <= tol).all()
        assert (state - last).abs().max() <= 1e-5
        only = ops.gated_block_step(proj[0], res[0], state, w)
        assert len(only) == 2


@gpu
def test_block_partial_gradients():
    """Only the state's gradient, only the output's, and no next norm."""
    gen = torch.Generator().manual_seed(3)
    T, B, H = 20, 2, 24
    proj, res = make(gen, T, B, 3 * H).cuda().requires_grad_(True), make(gen, T, B, H).cuda().requires_grad_(True)
    w = torch.ones(H, device='cuda')
    h0 = torch.zeros(H, device='cuda')
    out, last = ops.gated_block(proj, res, h0, w)
    g = torch.autograd.grad(last.sum(), proj, retain_graph=True)[0]
    x = proj.detach()[..., :2 * H].requires_grad_(True)
    _, last2 = ops.gated_scan(x, h0)
    assert torch.equal(g[..., :2 * H], torch.autograd.grad(last2.sum(), x)[0]) and not g[..., 2 * H:].any()
    gp, gr = torch.autograd.grad(out.sum(), [proj, res])
    assert torch.equal(gr, torch.ones_like(gr)) and torch.isfinite(gp).all()


@gpu
def test_block_on_any_strides():
    """Batch-first projections and residuals (whose rows have no one stride), column slices and expanded tensors: bit for bit
    what contiguous copies give, with gradients and without."""
    gen = torch.Generator().manual_seed(13)
    T, B, H = 45, 6, 20
    wide = make(gen, B, T, 3 * H + 8).cuda()
    res_b = make(gen, B, T, 2 * H).cuda()
    mask = (torch.rand(B, T, generator=gen) > 0.3).cuda().t()
    w, w2 = make(gen, H).cuda(), make(gen, 2 * H).cuda()[::2]
    h0 = make(gen, H, B).cuda().t()
    g = [make(gen, H).cuda().expand(T, B, H), make(gen, B, T, H).cuda().transpose(0, 1), make(gen, H, B).cuda().t()]
    for proj in (wide[..., 4:4 + 3 * H].transpose(0, 1), make(gen, 3 * H).cuda().expand(T, B, 3 * H)):
        res = res_b[..., ::2].transpose(0, 1)
        outs = []
        for fix in (lambda t: t, lambda t: t.contiguous()):
            args = [fix(t).detach() for t in (proj, res, h0, w, w2)]
            with torch.no_grad():
                found = list(ops.gated_block(*args[:4], next_weight=args[4], mask=fix(mask)))
            args = [a.requires_grad_(True) for a in args]
            got = ops.gated_block(*args[:4], next_weight=args[4], mask=fix(mask))
            found += list(got) + list(torch.autograd.grad(got, args, [fix(t) for t in g]))
            outs.append(found)
        for a, b in zip(*outs):
            assert torch.equal(a, b)


@gpu
def test_replayed_from_a_graph():
    """Forward and backward of a layer captured once and replayed on new inputs, with eager work between the replays:
    bit for bit the eager results."""
    gen = torch.Generator().manual_seed(4)
    T, B, H = 150, 4, 64
    proj, res = make(gen, T, B, 3 * H).cuda(), make(gen, T, B, H).cuda()
    h0, w, w2 = make(gen, H).cuda(), make(gen, H).cuda(), make(gen, H).cuda()
    g = make(gen, T, B, H).cuda()

    def work(p, r):
        p, r, hh, ww, nn = (t.detach().requires_grad_(True) for t in (p, r, h0, w, w2))
        out, n, last = ops.gated_block(p, r, hh, ww, next_weight=nn)
        return [out, n, last] + list(torch.autograd.grad([out, n], [p, r, hh, ww, nn], [g, g]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(proj, res)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work(proj, res)
    for k in range(3):
        proj.copy_(make(gen, T, B, 3 * H))
        res.copy_(make(gen, T, B, H))
        want = [t.clone() for t in work(proj, res)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


@gpu
def test_on_another_stream():
    gen = torch.Generator().manual_seed(12)
    x = make(gen, 300, 2, 64).cuda()
    want, _ = ops.gated_scan(x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got, _ = ops.gated_scan(x)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(want, got)


# ---- refusals (on the CPU too: every check of shapes and types comes before the device's) ---------------------------

Z = torch.zeros


@pytest.mark.parametrize('call', [
    lambda: ops.gated_scan(Z(4, 6)),
    lambda: ops.gated_scan(Z(4, 2, 5)),
    lambda: ops.gated_scan(Z(4, 2, 6, dtype=torch.float16)),
    lambda: ops.gated_scan(Z(4, 2, 6), Z(4)),
    lambda: ops.gated_scan(Z(4, 2, 6), mask=Z(2, 4)),
    lambda: ops.gated_scan_step(Z(2, 6), Z(2, 4)),
    lambda: ops.gated_scan_step(Z(2, 6), Z(2, 3).double()),
    lambda: ops.gated_scan_step(Z(2, 6), Z(3, 2).t()),
    lambda: ops.gated_scan_step(Z(2, 6), Z(2, 3), new_state=Z(1, 3)),
    lambda: ops.gated_scan_step(Z(2, 6, requires_grad=True), Z(2, 3)),
    lambda: ops.gated_scan_step(Z(2, 6), Z(2, 3), mask=Z(3)),
    lambda: ops.rms_norm(Z(2, 6), Z(5)),
    lambda: ops.rms_norm(Z(2, 6), Z(6).double()),
    lambda: ops.rms_norm(Z(2, 6, dtype=torch.float16), Z(6)),
    lambda: ops.rms_norm(Z(2, 6, dtype=BF16), Z(6), dtype=F32),
    lambda: ops.rms_norm(Z(2, 8193), Z(8193)),
    lambda: ops.rms_norm(Z(2, 0), Z(0)),
    lambda: ops.block_norm(Z(2, 6), Z(2, 5), Z(6)),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6), Z(6), gate=Z(2, 5)),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6), Z(6), gate=Z(2, 6, dtype=BF16)),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6, dtype=BF16), Z(6)),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6), None),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6), Z(6), scale=0.5),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6), Z(6), next_weight=Z(7)),
    lambda: ops.gated_block(Z(4, 2, 8), Z(4, 2, 3), None, Z(3)),
    lambda: ops.gated_block(Z(4, 2, 9), Z(4, 2, 3, dtype=BF16), None, Z(3)),
    lambda: ops.gated_block(Z(4, 2, 9), Z(4, 2, 3), Z(2), Z(3)),
    lambda: ops.gated_block_step(Z(2, 9), Z(2, 3), Z(2, 3), Z(3, requires_grad=True)),
    lambda: ops.gated_block_step(Z(2, 9), Z(2, 3), Z(3, 3), Z(3)),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize('call', [
    lambda: ops.gated_scan(Z(4, 2, 6)), lambda: ops.gated_scan_step(Z(2, 6), Z(2, 3)), lambda: ops.rms_norm(Z(2, 6), Z(6)),
    lambda: ops.block_norm(Z(2, 6), Z(2, 6), Z(6)), lambda: ops.gated_block(Z(4, 2, 9), Z(4, 2, 3), None, Z(3)),
    lambda: ops.gated_block_step(Z(2, 9), Z(2, 3), Z(2, 3), Z(3))])
def test_no_cpu_fallback(call):
    with pytest.raises(native.MdmmError):
        call()


@pytest.mark.parametrize('call', [
    lambda: ops.gated_scan(Z(1, 1, 2).expand(2 ** 31, 1, 2)), lambda: ops.gated_scan_step(Z(1, 2).expand(2 ** 31, 2), Z(1, 1)),
    lambda: ops.gated_block(Z(1, 1, 3).expand(2 ** 31, 1, 3), Z(1, 1, 1).expand(2 ** 31, 1, 1), None, Z(1))])
def test_dimensions_past_32_bits_are_refused(call):
    with pytest.raises(ValueError, match='2\\^31'):
        call()


def test_negative_batch_strides_are_refused_by_the_library():
    for field in ('gates_sb', 'g_gates_sb', 'mask_sb'):
        a = native.GatedScan()
        a.T, a.B, a.H, a.gates = 3, 2, 4, 64
        assert native.lib().mdmm_gated_scan_ws(a, 0) >= 0
        setattr(a, field, -8)
        assert native.lib().mdmm_gated_scan_ws(a, 0) < 0 and native.lib().mdmm_gated_scan_fwd(a, None) < 0


@pytest.mark.parametrize('module', ['recurrent', 'ortho', 'ops'])
def test_modules_import_in_any_order(module):
    """Each as the first module of a process."""
    subprocess.run([sys.executable, '-c', 'import mdmm.%s, mdmm.ops; mdmm.ops.gated_scan, mdmm.ops.orthogonalise' % module],
                   check=True, env=dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(native.__file__))), timeout=300)


@gpu
@pytest.mark.parametrize('H', [1, 2, 3, 4])
def test_narrow_rows_keep_their_gradients(H):
    """A row of one column is normalised to its sign: its gradient is eps r^3, what two nearly equal terms leave.  The inputs
    are exact, the arithmetic is 64-bit and only the stored gradients (and the fp32 slabs of the sums, 4 u of their terms'
    absolute sum) are rounded."""
    gen = torch.Generator().manual_seed(11)
    t = [make(gen, 300, H) for _ in range(5)] + [make(gen, H, mean=1.0, std=0.2) for _ in range(3)]
    y, res, gate, g_out, g_n, w, s, w2 = t
    cpu = [v.double().requires_grad_() for v in (y, res, w, gate, s, w2)]
    out = cpu[1] + cpu[4] * torch.nn.functional.silu(cpu[3]) * cpu[0] * (cpu[0].square().mean(-1, keepdim=True) + 1e-6).rsqrt() * cpu[2]
    n = out * (out.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * cpu[5]
    want = torch.autograd.grad([out, n], cpu, [g_out.double(), g_n.double()])
    dev = [v.cuda().requires_grad_() for v in (y, res, w, gate, s, w2)]
    got = torch.autograd.grad(ops.block_norm(dev[0], dev[1], dev[2], gate=dev[3], scale=dev[4], next_weight=dev[5]), dev,
                              [g_out.cuda(), g_n.cuda()])
    # terms of the sums: d_w = sum d_y-like terms p y r, bounded by |d_res s silu(g) y r| etc.
    r = (y.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    act = torch.nn.functional.silu(gate.double())
    terms = {2: want[1] * s.double() * act * y.double() * r, 4: want[1] * act * y.double() * r * w.double(),
             5: g_n.double() * out.detach() * (out.detach().square().mean(-1, keepdim=True) + 1e-6).rsqrt()}
    for i, (a, b) in enumerate(zip(got, want)):
        bound = 8 * U * terms[i].abs().sum(0) if i in terms else 2 * U * b.abs()
        assert ((a.cpu().double() - b).abs() <= bound + 1e-38).all(), (i, (a.cpu().double() - b).abs().max())


def dual(*shape, **kw):
    return torch.autograd.forward_ad.make_dual(Z(*shape, **kw), torch.ones(*shape, **kw))


@gpu
@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_is_refused(grad):
    """A tangent that went in and did not come out would be a wrong derivative: every operator raises."""
    w = torch.ones(3, device='cuda')
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for call in (lambda: ops.gated_scan(dual(4, 2, 6, device='cuda')),
                     lambda: ops.gated_scan(Z(4, 2, 6, device='cuda'), dual(3, device='cuda')),
                     lambda: ops.rms_norm(dual(2, 3, device='cuda'), w), lambda: ops.rms_norm(Z(2, 3, device='cuda'), dual(3, device='cuda')),
                     lambda: ops.block_norm(Z(2, 3, device='cuda'), dual(2, 3, device='cuda'), w),
                     lambda: ops.gated_block(dual(4, 2, 9, device='cuda'), Z(4, 2, 3, device='cuda'), None, w)):
            with pytest.raises(NotImplementedError):
                call()
        ops.gated_scan(Z(4, 2, 6, device='cuda'))              # (no tangent: as ever)


def test_forward_mode_is_refused_by_the_steps():
    with torch.autograd.forward_ad.dual_level():
        for call in (lambda: ops.gated_scan_step(dual(2, 6), Z(2, 3)), lambda: ops.gated_scan_step(Z(2, 6), dual(2, 3)),
                     lambda: ops.gated_block_step(Z(2, 9), dual(2, 3), Z(2, 3), Z(3))):
            with pytest.raises(ValueError):
                call()
