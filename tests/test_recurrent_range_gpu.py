"""The recurrent operators over the whole range of values and sizes: gates of any size, scans over several tiles."""
import pytest
import torch

from mdmm import native, ops
from test_recurrent_gpu import BF16, F32, U, close, make, scan_ref

gpu = pytest.mark.gpu
Z = torch.zeros
GATES = torch.tensor([-80.0, -60.0, -40.0, -20.0, -10.0, -5.0, -3.0, 0.5, 3.0, 10.0, 17.0, 30.0, 88.0, 1e2, 1e4, 3e7, 1e8, 1e12])


def gated_rows(H):
    gen = torch.Generator().manual_seed(31 + H)
    rows = 64
    gate = GATES[torch.randint(0, len(GATES), (rows, H), generator=gen)] * (1 + 0.01 * torch.rand(rows, H, generator=gen))
    y, w = make(gen, rows, H), make(gen, H, std=0.1, mean=1.0)
    g_out = torch.where(torch.rand(rows, H, generator=gen) > 0.5, 1.0, -1.0)
    return rows, gate, y, w, g_out, y.double() * torch.rsqrt(y.double().square().mean(-1, keepdim=True) + 1e-6) * w.double()


# The gate's factor 6 u (its exponential, the sum, the reciprocal, two products), r 14 u (a sum of H squares in pieces, at most
# 20 u of the mean, half of it in its root, and the root's own 4), four products; twice that is allowed
TOL = 2 * (6 + 14 + 4) * U


@gpu
@pytest.mark.parametrize('H', [3, 100, 256, 700])
def test_gates_of_any_size(H):
    """silu(g) to a few units of its own size wherever g lies: an output without a residual is a product."""
    rows, gate, y, w, _, u = gated_rows(H)
    want = gate.double() * torch.sigmoid(gate.double()) * u
    out = ops.block_norm(y.cuda(), Z(rows, H).cuda(), w.cuda(), gate=gate.cuda())
    assert ((out.cpu().double() - want).abs() <= TOL * want.abs() + 1e-37).all()
    # the step form: a state that the masked step leaves as it is
    proj = torch.cat([Z(rows, 2 * H), gate], -1).cuda()
    out, _ = ops.gated_block_step(proj, Z(rows, H).cuda(), y.cuda(), w.cuda(), mask=Z(rows, dtype=torch.bool).cuda())
    assert ((out.cpu().double() - want).abs() <= TOL * want.abs() + 1e-37).all()


@gpu
@pytest.mark.parametrize('H', [3, 100, 256, 700])
def test_slopes_of_any_gate(H):
    """The gate's gradient g_out u silu'(g) to a few units of its own size.  silu'(g) = a (1 + g k) adds u (1 + |g k|) /
    |1 + g k| on the way to its zero at g = -1.28, from which these gates keep away."""
    rows, gate, y, w, g_out, u = gated_rows(H)
    g64 = gate.double()
    k = torch.sigmoid(-g64)
    want = g_out.double() * u * torch.sigmoid(g64) * (1 + g64 * k)
    lost = (1 + (g64 * k).abs()) / (1 + g64 * k).abs()
    gd = gate.cuda().requires_grad_(True)
    got = torch.autograd.grad(ops.block_norm(y.cuda(), Z(rows, H).cuda(), w.cuda(), gate=gd), gd, g_out.cuda())[0]
    assert ((got.cpu().double() - want).abs() <= TOL * (1 + lost) * want.abs() + 1e-37).all()


@gpu
@pytest.mark.parametrize('T,B,H', [(1, 3, 20), (64, 2, 12), (40, 3, 33)])
def test_no_states_are_written_where_none_are_asked_for(T, B, H):
    """A C caller with one buffer for everything: up to 64 steps mdmm_gated_scan_states is 0, and what lies at `states` is
    neither written nor read."""
    gen = torch.Generator().manual_seed(T)
    x, g = make(gen, T, B, 2 * H).cuda(), make(gen, T, B, H).cuda()
    xd = x.clone().requires_grad_(True)
    want = ops.gated_scan(xd)[0]
    want_g = torch.autograd.grad(want, xd, g)[0]
    room = torch.full((4 * B * H,), 7.0, device='cuda')
    h, g_x = torch.empty(T, B, H, device='cuda'), torch.empty_like(x)
    a = native.GatedScan()
    a.T, a.B, a.H = T, B, H
    a.gates, a.gates_st, a.gates_sb, a.h, a.states = x.data_ptr(), 2 * B * H, 2 * H, h.data_ptr(), room.data_ptr()
    assert native.lib().mdmm_gated_scan_states(a) == 0 and native.lib().mdmm_gated_scan_ws(a, 0) == 0
    stream = torch.cuda.current_stream().cuda_stream
    native.check(native.lib().mdmm_gated_scan_fwd(a, stream), 'mdmm_gated_scan_fwd')
    a.g_h, a.g_gates, a.g_gates_st, a.g_gates_sb = g.data_ptr(), g_x.data_ptr(), 2 * B * H, 2 * H
    native.check(native.lib().mdmm_gated_scan_bwd(a, stream), 'mdmm_gated_scan_bwd')
    assert torch.equal(room, torch.full_like(room, 7.0)) and torch.equal(h, want) and torch.equal(g_x, want_g)


def test_new_states_beside_inputs_are_not_refused():
    flat = Z(64)
    a, p, c = flat[:6].view(2, 3), flat[:18].view(2, 9), flat[20:26].view(2, 3)
    for call in (lambda: ops.gated_block_step(Z(2, 9), Z(2, 3), a, Z(3), new_state=a), lambda: ops.gated_scan_step(Z(2, 6), a, new_state=c),
                 lambda: ops.gated_scan_step(p[:, :6], c, new_state=c)):
        with pytest.raises(native.MdmmError):          # (the device's refusal, which comes last)
            call()


def step_structs(B=2, H=4):
    """A time step on made-up addresses, for refusals that come before any launch."""
    a, p = native.GatedScan(), native.BlockNorm()
    a.T, a.B, a.H = 1, B, H
    a.gates, a.gates_sb, a.h0, a.h0_sb, a.h_last, a.mask, a.mask_sb = 0x10000, 3 * H, 0x20000, H, 0x30000, 0x40000, 1
    p.rows, p.H, p.eps = B, H, 1e-6
    p.res, p.res_st, p.out, p.out_st, p.w, p.scale, p.w_next = 0x50000, H, 0x60000, H, 0x70000, 0x80000, 0x90000
    p.n, p.n_st, p.gate, p.gate_st = 0xa0000, H, 0x10000 + 8 * H, 3 * H
    return a, p


@pytest.mark.parametrize('at', ['gates', 'gates + 72', 'h0 + 16', 'h0 - 16', 'mask', 'mask - 31', 'res', 'res + 31', 'w', 'scale + 8',
                                'w_next - 28'])
def test_new_states_on_top_of_inputs_are_refused(at):
    name, _, off = at.partition(' ')
    off = int(off.replace(' ', '') or 0)
    a, p = step_structs()
    a.h_last = (getattr(a, name) if hasattr(a, name) else getattr(p, name)) + off
    assert native.lib().mdmm_gated_block_step(a, p, None) == -4
    if hasattr(a, name):
        a.h = 0xb0000
        assert native.lib().mdmm_gated_scan_fwd(a, None) == -4


def test_longer_scans_in_place_are_refused():
    a, _ = step_structs()
    a.T, a.h, a.h_last = 2, 0xb0000, a.h0
    assert native.lib().mdmm_gated_scan_fwd(a, None) == -4


@gpu
def test_steps_in_place_and_beside():
    """In place, into another tensor and into a neighbour within one buffer: the same; on top of an input: an error."""
    gen = torch.Generator().manual_seed(3)
    H = 4
    proj, res, w = make(gen, 2, 3 * H).cuda(), make(gen, 2, H).cuda(), torch.ones(H, device='cuda')
    start = make(gen, 2, H).cuda()
    want_out, want = ops.gated_block_step(proj, res, start, w)
    both = torch.zeros(4, H, device='cuda')
    for state, new in ((start.clone(), None), (both[:2].copy_(start), both[2:])):
        out, got = ops.gated_block_step(proj, res, state, w, new_state=state if new is None else new)
        assert torch.equal(out, want_out) and torch.equal(got, want)
    both[:2].copy_(start)
    for args, new in (((res, start), res), ((both[:2], both[:2]), both[:2]), ((res, both[:2]), both[1:3])):
        with pytest.raises(native.MdmmError, match='shares memory'):
            ops.gated_block_step(proj, args[0], args[1], w, new_state=new)
    gates = make(gen, 2, 2 * H).cuda()
    with pytest.raises(native.MdmmError, match='shares memory'):
        ops.gated_scan_step(gates, start, new_state=gates.view(4, H)[1:3])


@gpu
@pytest.mark.parametrize('T,B,H', [(101, 64, 1024), (301, 8, 2048), (333, 40, 515)])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('reverse', [False, True])
def test_scan_over_several_tiles(T, B, H, dtype, reverse):
    """Workgroups that walk over several tiles of time, alone over it and with it split (a ragged last split too)."""
    gen = torch.Generator().manual_seed(T + B)
    gates = torch.cat([make(gen, T, B, H, std=1.5, mean=2.0), make(gen, T, B, H)], -1).to(dtype)
    m = torch.rand(T, B, generator=gen) > 0.2
    h0, g_h, g_last = make(gen, H), make(gen, T, B, H, dtype=dtype), make(gen, B, H)
    want = scan_ref(gates, h0, m, reverse, g_h, g_last)
    x, hd = gates.cuda().requires_grad_(True), h0.cuda().requires_grad_(True)
    h, last = ops.gated_scan(x, hd, mask=m.cuda(), reverse=reverse)
    grads = torch.autograd.grad([h, last], [x, hd], [g_h.cuda(), g_last.cuda()])
    for got, name in ((h, 'h'), (last, 'last'), (grads[0], 'gates'), (grads[1], 'h0')):
        close(got, want[name], name)


@gpu
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_masked_steps_get_zero_gradients_whatever_comes_in(bad):
    """The gradient of a state that a masked step left as it is belongs to the states before it: f and c of that step get
    zeros, also where it is not finite."""
    gen = torch.Generator().manual_seed(6)
    T, B, H = 70, 2, 6
    x, g = make(gen, T, B, 2 * H).cuda().requires_grad_(True), make(gen, T, B, H).cuda()
    mask = torch.ones(T, B, dtype=torch.bool, device='cuda')
    mask[:3, 0] = False
    mask[40, 1] = False
    h, _ = ops.gated_scan(x, mask=mask)
    want = torch.autograd.grad(h, x, g, retain_graph=True)[0]
    g[2, 0] = bad                          # (no step of this sequence lies before it)
    g[40, 1] = bad
    got = torch.autograd.grad(h, x, g)[0]
    assert torch.equal(got[:, 0], want[:, 0]) and not got[:3, 0].any()
    assert torch.equal(got[40:, 1], want[40:, 1]) and not got[40, 1].any() and not torch.isfinite(got[:40, 1]).any()
