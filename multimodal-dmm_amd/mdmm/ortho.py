"""Orthogonalised updates of weight matrices by Newton-Schulz products (csrc/ortho.hip).  Public as mdmm.ops.orthogonalise;
harness.FlatMuon is the optimizer made of it."""
import ctypes as C

import torch

from . import native

# X <- a X + (b A + c A^2) X, A = X X^T: these take every singular value in (0, 1] to about 1 (between 0.7 and 1.2) in five
# steps, the slope a at 0 as steep as that allows -- the values of the Muon optimizer's published description
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


# the kernels' fp16 plane pairs hold X and A up to 4, P = b A + c A^2 up to 16; a step count that no iteration needs
MAX_X, MAX_P, MAX_STEPS = 1.95, 15.5, 1000
MAX_SIDE = 65536


def _bounded(steps, a, b, c):
    """Whether the singular values and P's, from (0, 1] on, stay within what the kernels hold."""
    top = 1.0
    for _ in range(steps):
        ends = [top * top]                          # u = s^2: the end, p's slope and P's slope at zero
        if c:
            ends.append(-b / (2.0 * c))
            root = 9.0 * b * b - 20.0 * a * c
            if root >= 0.0:
                ends += [(-3.0 * b + sign * root ** 0.5) / (10.0 * c) for sign in (1.0, -1.0)]
        elif b:
            ends.append(-a / (3.0 * b))
        ends = [u for u in ends if 0.0 <= u <= top * top]
        new = max([u ** 0.5 * abs(a + b * u + c * u * u) for u in ends])
        if not (top <= MAX_X and max([abs(b * u + c * u * u) for u in ends]) <= MAX_P):
            return False
        if not new > top:
            return new == new
        top = new
    return True


def as_matrix(t):
    """A parameter's (rows, cols) view: leading dimension x the rest, as a convolution's kernels are applied."""
    return t if t.dim() == 2 else t.reshape(t.shape[0], -1)


def launch(items, steps, eps, coefficients, src_bf16, dst_bf16, momentum=0.0, nesterov=False, update=False, lr=0.0, lr_dev=None,
           decay=0.0, device=None):
    """items: (src, mom or None, dst, gain) with (rows, cols) unit-column-stride tensors; MDMM_ORTHO_MAX to a call."""
    for k in range(0, len(items), native.ORTHO_MAX):
        part = items[k:k + native.ORTHO_MAX]
        a = native.Ortho()
        a.n, a.steps, a.src_bf16, a.dst_bf16 = len(part), steps, int(src_bf16), int(dst_bf16)
        a.nesterov, a.update, a.eps, a.momentum, a.decay, a.lr = int(nesterov), int(update), eps, momentum, decay, lr
        a.ca, a.cb, a.cc = coefficients
        a.lr_dev = ops._ptr(lr_dev)
        for it, (src, mom, dst, gain) in zip(a.item, part):
            it.src, it.mom, it.dst, it.gain = src.data_ptr(), ops._ptr(mom), dst.data_ptr(), gain
            it.rows, it.cols = src.shape
            it.src_ld, it.dst_ld = max(src.stride(0), src.shape[1]), max(dst.stride(0), dst.shape[1])
        nbytes = native.lib().mdmm_ortho_ws(C.byref(a))
        if nbytes < 0:
            native.check(nbytes, 'mdmm_ortho_ws')
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        a.ws = ws.data_ptr()
        ops._call('mdmm_ortho', C.byref(a), tag='ortho[%d]' % len(part))


def orthogonalise(mats, steps=5, eps=1e-7, coefficients=COEFFICIENTS):
    """The nearest-orthogonal direction of every matrix of a list, U V^T of M = U S V^T approximately, by `steps`
    Newton-Schulz steps on M / (|M|_F + eps), accurate to a few roundings of fp32: with shorter sides of up to 128 the matrices
    are fp32, beyond kept to 22 to 23 bits instead of 24 with better sums (the error of fp32 products by the library: 0.3 to 0.8
    of it, up to 1.3 for shorter sides below ten).  Matrices of one type and size class share the launches, 24 to a call.

    mats: fp32 or bf16 tensors of two or more dimensions (more than two: leading dimension x the rest), either side the
    longer, at most 65536.  coefficients: (a, b, c) of X <- a X + (b A + c A^2) X, A = X X^T, such that singular values in
    (0, 1] stay below 1.95 (refused otherwise).  -> a list of contiguous tensors of their shapes and types.  No gradient: a
    matrix that wants one is refused."""
    mats = [mats] if torch.is_tensor(mats) else list(mats)
    if int(steps) != steps or not 0 <= steps <= MAX_STEPS:
        raise ValueError('orthogonalise: a number of steps, 0 to %d, got %r' % (MAX_STEPS, steps))
    if len(coefficients) != 3:
        raise ValueError('orthogonalise: three coefficients, got %r' % (coefficients,))
    coefficients = tuple(float(c) for c in coefficients)
    if coefficients != COEFFICIENTS and not _bounded(int(steps), *coefficients):
        raise ValueError('orthogonalise: singular values must stay below %g and those of b A + c A^2 below %g, with %r they do not'
                         % (MAX_X, MAX_P, coefficients))
    if not mats:
        return []
    for m in mats:
        if m.dim() < 2:
            raise ValueError('orthogonalise: matrices, got shape %s' % (tuple(m.shape),))
        if recurrent._grad_wanted(m):
            raise ValueError('orthogonalise has no gradient: call it under torch.no_grad(), or on detached matrices')
        if m.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError('orthogonalise: fp32 or bf16 matrices, got %s' % m.dtype)
        if m.shape[0] > MAX_SIDE or m.numel() > MAX_SIDE * max(m.shape[0], 1):
            raise ValueError('orthogonalise: at most %d rows and columns, got %s' % (MAX_SIDE, tuple(m.shape)))
    for m in mats:
        ops._need_gpu(m)
        if m.device != mats[0].device:
            raise ValueError('orthogonalise: matrices on %s and %s' % (mats[0].device, m.device))
    dev = mats[0].device
    with torch.no_grad(), torch.cuda.device(dev):
        outs = [torch.empty(m.shape, device=dev, dtype=m.dtype) for m in mats]
        for dtype in (torch.float32, torch.bfloat16):
            items = []
            for m, o in zip(mats, outs):
                if m.dtype == dtype and m.numel():
                    src = as_matrix(m.detach())
                    if src.stride(1) != 1 or (src.shape[0] > 1 and src.stride(0) < src.shape[1]):
                        src = src.contiguous()
                    items.append((src, None, as_matrix(o), 1.0))
            if items:
                bf = dtype == torch.bfloat16
                launch(items, int(steps), float(eps), coefficients, bf, bf, device=dev)
    return outs


from . import ops, recurrent  # noqa: E402  (last: ops re-exports this module's functions, whichever of the two is imported first)
