"""8-bit checkpoints, complex group norm and class scores against plain implementations in 64 bits on the CPU.

u = 2^-24 is the rounding of a float32 operation (half a step, relative).  Tolerances are worst-case counts of such roundings
along the formula; the comment at each says which."""
import gc

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _features(n, cols, seed, parts=2):
    """Rows of different magnitude, channels with offsets: what a convolution hands on."""
    g = _gen(seed)
    x = torch.randn(n, parts, cols, generator=g) * torch.exp(0.7 * torch.randn(n, 1, 1, generator=g))
    return x + torch.randn(1, parts, cols, generator=g)


# ---------------------------------------------------------------------------------------------
# 8-bit checkpoints
# ---------------------------------------------------------------------------------------------
def _restored(x):
    """The format by its definition, 64 bits on the host: x float32 [..., m] -> the values a checkpoint of it restores."""
    a = x.double().numpy()
    m = a.shape[-1]
    out = np.empty_like(a)
    for c in range(0, m, 32):
        b = a[..., c:c + 32]
        ok = np.isfinite(b).all(-1, keepdims=True)
        b = np.where(ok, b, 0.0)
        top = np.abs(b).max(-1, keepdims=True)
        f, p = np.frexp(top)
        s = np.where(np.rint(f * 128) > 127, p - 6, p - 7)
        step = np.ldexp(1.0, np.clip(s, -110, 121))
        out[..., c:c + 32] = np.where(ok, np.clip(np.rint(b / step), -127, 127) * step, np.nan)
    return out


def _same(got, want):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.array_equal(got, want, equal_nan=True), 'max off by %g' % np.nanmax(np.abs(got - want))


@pytest.mark.parametrize('n,m', [(0, 5), (1, 1), (1, 33), (2, 4), (3, 32), (5, 31), (17, 48), (129, 30), (64, 1000), (4, 4100), (3001, 7),
                                 (1000, 128)])
def test_checkpoint_restores_the_nearest_value_of_its_format(n, m):
    from magnet_amd.checkpoint import Checkpoint8
    x = _features(n, m, seed=n * 7 + m)
    ck = Checkpoint8.store(x.to(DEV))
    assert ck.codes.shape == (2 * n, -(-m // 32) * 32) and ck.scales.shape == (-(-m // 32), -(-2 * n // 8) * 8)
    assert ck.nbytes() == ck.codes.numel() + ck.scales.numel()
    _same(ck.restore(), _restored(x))
    # the bytes behind the matrix are what the format says
    assert bool((ck.codes[:, m:] == 128).all()) and bool((ck.scales[:, 2 * n:] == 0).all())


def test_checkpoint_of_awkward_values():
    from magnet_amd.checkpoint import Checkpoint8
    x = torch.zeros(12, 2, 64)
    x[1] = torch.linspace(-1e-38, 1e-38, 64)                       # around the smallest normal number
    x[2] = torch.linspace(-3e-45, 3e-45, 64)                       # subnormal
    x[3] = torch.linspace(-3.4028234e38, 3.4028234e38, 64)         # up to the largest
    x[4, 0, :32] = 127.5 / 128 * torch.linspace(-1, 1, 32)         # the largest rounds to 128: one more step of scale
    x[4, 0, 32:] = float(np.nextafter(np.float32(127.5 / 128), np.float32(0))) * torch.linspace(-1, 1, 32)
    x[5] = (torch.arange(64) - 31.5) / 64.0                        # ties
    x[5, :, 0] = x[5, :, 32] = 100.0
    x[6, 0, 3] = float('nan')
    x[6, 1, 40] = float('inf')
    x[7, 0, 40] = -float('inf')
    x[7, 1] = -0.0
    x[8] = 2.0 ** -110 * (torch.arange(64) - 31.5)                 # the smallest scale
    x[9] = 2.0 ** torch.arange(-32, 32).float()
    x[10, 0, 5] = 1e30
    x[10, 0, 6] = 1e-30
    _same(Checkpoint8.store(x.to(DEV)).restore(), _restored(x))


def test_checkpoint_error_is_half_a_step():
    from magnet_amd.checkpoint import Checkpoint8
    x = _features(700, 96, seed=3)
    got = Checkpoint8.store(x.to(DEV)).restore().double().cpu().view(700, 2, 3, 32)
    x = x.double().view(700, 2, 3, 32)
    # top = f 2^p with f in [1/2, 127.5/128): half a step is 2^(p-8) <= top / 128; from 127.5/128 on it is 2^(p-7) <= top / 127.5
    top = x.abs().amax(-1, keepdim=True)
    assert bool(((got - x).abs() <= top / 127.5).all())
    f, p = torch.frexp(top)
    assert bool(((got - x).abs() <= torch.ldexp(torch.ones_like(f), torch.where(f < 127.5 / 128, p - 8, p - 7))).all())


@pytest.mark.parametrize('f', [8, 30, 32])
def test_checkpoint_takes_strided_input_and_output(f):
    """One order of a side-by-side block, a column slice that starts off 16 bytes, a transposed layout; and a restore into one."""
    from magnet_amd.checkpoint import Checkpoint8
    block = _features(41, 3 * f, seed=f).to(DEV).view(41, 2, 3, f)
    for x in (block[:, :, 1, :], block.view(41, 2, 3 * f)[:, :, 1:f], block[:, :, 2, :].flip(0), block[:, :, 0, :].transpose(0, 1).contiguous().transpose(0, 1),
              block[:, :, 0, :].transpose(1, 2).contiguous().transpose(1, 2), block[:1, :, 0, :].expand(9, 2, f)):
        ck = Checkpoint8.store(x)
        _same(ck.restore(), _restored(x.cpu().contiguous()))
        out = torch.full((x.size(0), 2, 2, x.size(2)), 7.0, device=DEV)
        ck.restore(out=out[:, :, 1, :])
        _same(out[:, :, 1, :], _restored(x.cpu().contiguous()))
        assert bool((out[:, :, 0, :] == 7.0).all())                # nothing beside it is written
    ck = Checkpoint8.store(block)
    assert ck.restore().shape == block.shape
    _same(ck.restore().view(41, 2, 3 * f), _restored(block.view(41, 2, 3 * f).cpu()))


def _gram_check(got, a, g):
    """a [R, m], g [R, k] float64.  A product of a 7-bit and a 24-bit number is three exact bf16 products; they and the slab's
    sum are added in float32: at most 3 R additions on the way to a result, each off by u of a partial sum that is at most
    sum |a g|; the join over slabs is in 64 bits, the last rounding adds u."""
    want, most = a.t() @ g, a.abs().t() @ g.abs()
    err = (got.double().cpu() - want).abs()
    bound = (3 * a.size(0) + 2) * U * most + 1e-300
    assert bool((err <= bound).all()), float((err / bound).max())
    # and the framework's bar for float32 results
    assert float(err.max()) <= 1e-5 * float(want.abs().max()) + 1e-30


@pytest.mark.parametrize('n,m,k', [(1, 1, 1), (3, 5, 2), (4, 32, 32), (31, 33, 31), (100, 48, 16), (257, 130, 65), (1025, 256, 128),
                                   (640, 300, 129), (700, 512, 257), (5000, 96, 100), (20000, 64, 64), (9999, 385, 33), (3000, 1, 200),
                                   (3000, 200, 1)])
def test_gram_of_a_checkpoint(n, m, k):
    from magnet_amd.checkpoint import Checkpoint8
    x = _features(n, m, seed=n + m)
    g = torch.randn(n, 2, k, generator=_gen(k)) * (torch.rand(n, 1, k, generator=_gen(k + 1)) < 0.5) / n
    got = Checkpoint8.store(x.to(DEV)).gram(g.to(DEV))
    assert got.shape == (m, k) and got.dtype == torch.float32
    _gram_check(got, torch.from_numpy(_restored(x)).view(2 * n, m), g.double().view(2 * n, k))
    assert torch.equal(got, Checkpoint8.store(x.to(DEV)).gram(g.to(DEV)))          # the same result every time


def test_gram_of_nothing_and_of_awkward_gradients():
    from magnet_amd.checkpoint import Checkpoint8
    assert torch.equal(Checkpoint8.store(torch.zeros(0, 2, 6, device=DEV)).gram(torch.zeros(0, 2, 3, device=DEV)).cpu(), torch.zeros(6, 3))
    n, m, k = 333, 70, 40
    x = _features(n, m, seed=1)
    a = torch.from_numpy(_restored(x)).view(2 * n, m)
    ck = Checkpoint8.store(x.to(DEV))
    wide = torch.randn(n, 2, 3, k, generator=_gen(2))
    for g in (wide[:, :, 1, :], wide.view(n, 2, 3 * k)[:, :, 1:k + 1], wide[:, :, 2, :].transpose(0, 1).contiguous().transpose(0, 1),
              torch.tensor(0.25).expand(n, 2, k), wide[:1, :, 0, :].expand(n, 2, k)):
        gd = g.to(DEV) if 0 in g.stride() else torch.empty_strided(g.size(), g.stride(), device=DEV).copy_(g)
        _gram_check(ck.gram(gd), a, g.double().reshape(2 * n, k))
    # the gradient of a mean over 10^9 values, and one next to the largest float
    for scale in (1e-18, 1e-30, 1e30):
        g = wide[:, :, 0, :].contiguous() * scale
        _gram_check(ck.gram(g.to(DEV)) / scale, a, g.double().reshape(2 * n, k) / scale)
    # all orders of a block at once, as the GEMM-first convolution has them
    _gram_check(ck.gram(wide.to(DEV)), a, wide.double().reshape(2 * n, 3 * k))
    # a block that is not finite reaches its 32 columns and no others; a gradient that is not, its column
    x[5, 0, 40] = float('inf')
    got = Checkpoint8.store(x.to(DEV)).gram(wide[:, :, 0, :].to(DEV)).cpu()
    assert bool(torch.isnan(got[32:64]).all()) and not bool(torch.isnan(got[:32]).any()) and not bool(torch.isnan(got[64:]).any())
    g = wide[:, :, 0, :].clone()
    g[7, 1, 3] = float('nan')
    got = ck.gram(g.to(DEV)).cpu()
    assert bool(torch.isnan(got[:, 3]).all()) and not bool(torch.isnan(got[:, :3]).any()) and not bool(torch.isnan(got[:, 4:]).any())


def test_checkpoint_whose_offsets_pass_32_bits():
    """2.6 G codes: rows at the far end are stored, restored and summed where they belong."""
    from magnet_amd.checkpoint import Checkpoint8
    n, m = 5_100_000, 256
    x = torch.zeros(n, 2, m, device=DEV)
    rows = torch.tensor([0, 1, 2_097_151, 2_097_152, 4_194_303, 4_194_304, n - 2, n - 1])
    part = _features(len(rows), m, seed=9)
    x[rows.to(DEV)] = part.to(DEV)
    ck = Checkpoint8.store(x)
    assert ck.codes.numel() > 2 ** 31
    g = torch.zeros(n, 2, 8, device=DEV)
    gp = torch.randn(len(rows), 2, 8, generator=_gen(4))
    g[rows.to(DEV)] = gp.to(DEV)
    want = torch.from_numpy(_restored(part)).view(-1, m)
    _gram_check(ck.gram(g), want, gp.double().view(-1, 8))
    del g
    x.fill_(5.0)
    back = ck.restore(out=x)
    _same(back[rows.to(DEV)], want.view(-1, 2, m).numpy())
    sums = back.abs().sum(2).cpu().double()                        # of each row: the others are zeros
    assert float(sums.sum()) == pytest.approx(float(want.abs().sum()), rel=1e-5)


def test_checkpoint_refusals():
    from magnet_amd import MagnetHipError
    from magnet_amd.checkpoint import Checkpoint8
    ck = Checkpoint8.store(torch.zeros(6, 2, 40, device=DEV))
    codes, scales = ck.codes, ck.scales
    for call in (lambda: ck.gram(torch.zeros(5, 2, 3, device=DEV)), lambda: ck.gram(torch.zeros(6, 2, 0, device=DEV)),
                 lambda: ck.gram(torch.zeros(6, 2, 3)), lambda: ck.gram(torch.zeros(6, 2, 3, device=DEV, dtype=torch.float64)),
                 lambda: ck.restore(out=torch.zeros(6, 2, 41, device=DEV)), lambda: Checkpoint8.store(torch.zeros(6, 2, 0, device=DEV)),
                 lambda: Checkpoint8.store(torch.zeros(6, 2, 4, device=DEV, dtype=torch.bfloat16)),
                 lambda: Checkpoint8(codes[:-1], scales, (6, 2, 40)).restore(), lambda: Checkpoint8(codes, scales[:1], (6, 2, 40)).restore(),
                 lambda: Checkpoint8(codes, scales, (6, 2, 65)).restore(), lambda: Checkpoint8(codes.int(), scales, (6, 2, 40)).restore(),
                 lambda: Checkpoint8(codes, scales.cpu(), (6, 2, 40)).restore(), lambda: Checkpoint8(codes, scales, (7, 2, 40)).gram(torch.zeros(7, 2, 3, device=DEV))):
        with pytest.raises(MagnetHipError):
            call()


# ---------------------------------------------------------------------------------------------
# complex group norm
# ---------------------------------------------------------------------------------------------
def _norm_reference(x, groups, w, b, sizes, eps, relu, g, held=None):
    """64 bits, graph by graph: result, gradients of x, w, b, and the sums of magnitudes their tolerances need.  `held`: the
    values that stand for x in the backward pass."""
    n, _, f = x.shape
    out, dx, tol_out, tol_dx = (torch.zeros(n, 2, f, dtype=torch.float64) for _ in range(4))
    dw, db, mag_w, mag_b = (torch.zeros(f, dtype=torch.float64) for _ in range(4))
    at = 0
    for k in sizes:
        s = slice(at, at + k)
        at += k
        if k == 0:
            continue
        z = torch.complex(x[s, 0].double(), x[s, 1].double()).view(k, groups, -1)
        mean = z.mean((0, 2), keepdim=True)
        sd = torch.sqrt((z - mean).abs().square().mean((0, 2), keepdim=True) + eps)
        zn = ((z - mean) / sd).view(k, f)
        y = zn * w + torch.complex(b, b)
        gate = (y.real >= 0).double() if relu else torch.ones_like(y.real)
        out[s, 0], out[s, 1] = y.real * gate, y.imag * gate
        tol_out[s, 0], tol_out[s, 1] = (zn.real * w).abs() + b.abs(), (zn.imag * w).abs() + b.abs()
        if g is None:
            continue
        if held is not None:
            zn = ((torch.complex(held[s, 0], held[s, 1]).view(k, groups, -1) - mean) / sd).view(k, f)
        dy = torch.complex(g[s, 0].double(), g[s, 1].double()) * gate
        inner = (dy * zn.conj()).real
        mags = dy.real.abs() * zn.real.abs() + dy.imag.abs() * zn.imag.abs()
        dw += inner.sum(0)
        db += (dy.real + dy.imag).sum(0)
        mag_w += mags.sum(0)
        mag_b += (dy.real.abs() + dy.imag.abs()).sum(0)
        dz = (dy * w).view(k, groups, -1)
        pull = (inner * w).view(k, groups, -1).mean((0, 2), keepdim=True)
        d = ((dz - dz.mean((0, 2), keepdim=True) - zn.view(k, groups, -1) * pull) / sd).view(k, f)
        dx[s, 0], dx[s, 1] = d.real, d.imag
        flat = torch.complex(dz.real.abs(), dz.imag.abs()).mean((0, 2), keepdim=True)
        along = (mags * w.abs()).view(k, groups, -1).mean((0, 2), keepdim=True)
        for p, (v, q, fl) in enumerate(((zn.real, dz.real, flat.real), (zn.imag, dz.imag, flat.imag))):
            tol_dx[s, p] = ((q.abs() + fl + v.view(k, groups, -1).abs() * along) / sd).view(k, f)
    return out, dx, dw, db, tol_out, tol_dx, mag_w, mag_b


def _off_the_gate(x, groups, w, b, sizes, eps):
    """Moves values whose gate hangs on a rounding (|Re y| < 1e-4) off it: x float32 [N, 2, F], in place."""
    at = 0
    for k in sizes:
        if k:
            z = torch.complex(x[at:at + k, 0].double(), x[at:at + k, 1].double()).view(k, groups, -1)
            mean = z.mean((0, 2), keepdim=True)
            sd = torch.sqrt((z - mean).abs().square().mean((0, 2), keepdim=True) + eps)
            y = ((z - mean) / sd).view(k, -1) * w + torch.complex(b, b)
            x[at:at + k, 0] += (0.05 * sd.expand_as(z).reshape(k, -1) * (y.real.abs() < 1e-4)).float()
        at += k
    return x


def _close(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), '%s: %g of its bound' % (what, float((err / bound).max()))


NORM_CASES = [
    # nodes, feats, groups, sizes of the graphs (None: one), relu, rows behind the last graph
    (1, 1, 1, None, False, 0), (1, 8, 2, None, True, 0), (2, 3, 3, None, True, 0), (5, 4, 1, None, False, 0), (63, 30, 5, None, True, 0),
    (64, 32, 4, None, True, 0), (257, 16, 4, None, True, 0), (2500, 16, 4, None, True, 0), (1000, 128, 8, None, True, 0),
    (300, 260, 13, None, True, 0), (130, 600, 3, None, False, 0), (50, 1028, 4, None, True, 0), (40, 257, 257, None, True, 0),
    (30, 12, 2, (10, 0, 7, 13), True, 0), (30, 12, 3, (0, 0, 30), False, 0), (33, 7, 7, (1, 1, 31, 0), True, 0),
    (4100, 20, 5, (4000, 1, 99), True, 0), (100, 8, 2, (40, 20), True, 40), (70, 6, 1, (0, 0), False, 70),
    (900, 24, 2, tuple([3] * 299 + [3]), True, 0),
]


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('n,f,groups,sizes,relu,behind', NORM_CASES)
def test_group_norm_and_its_gradients(n, f, groups, sizes, relu, behind, bits):
    from magnet_amd.layer.norm import complex_group_norm
    x = _features(n, f, seed=n + f)
    w = 0.5 + torch.rand(f, generator=_gen(f))
    b = torch.rand(f, generator=_gen(f + 1)) - 0.3
    every = [n] if sizes is None else list(sizes)
    assert sum(every) + behind == n
    x = _off_the_gate(x, groups, w.double(), b.double(), every, 1e-5) if relu else x
    g = torch.randn(n, 2, f, generator=_gen(5))
    ptr = None if sizes is None else torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int64, device=DEV)
    held = torch.from_numpy(_restored(x)) if bits == 8 else None
    out, dx, dw, db, tol_out, tol_dx, mag_w, mag_b = _norm_reference(x, groups, w.double(), b.double(), every, 1e-5, relu, g, held)
    xd, wd, bd = (t.to(DEV).requires_grad_() for t in (x, w, b))
    y = complex_group_norm(xd, groups, wd, bd, graph_ptr=ptr, relu=relu, checkpoint_bits=bits)
    y.backward(g.to(DEV))
    # z - m, 1/sd, their product with w and the addition of b: 5 roundings; the mean's second float and the 64-bit statistics
    # add less than one
    _close(y.detach(), out, 8 * U * tol_out + 1e-300, 'result')
    # xh and dxh: 4 roundings each, the two differences and the last product 3, the means (of terms with up to 5) 5 more
    _close(xd.grad, dx, 20 * U * tol_dx + 1e-300, 'dx')
    # terms with up to 6 roundings, added in 64 bits
    _close(wd.grad, dw, 8 * U * mag_w + 1e-300, 'dweight')
    _close(bd.grad, db, 4 * U * mag_b + 1e-300, 'dbias')
    if behind:
        assert not bool(y[n - behind:].any()) and not bool(xd.grad[n - behind:].any())


def test_group_norm_far_from_zero_and_without_parameters():
    """A mean 10^4 deviations from 0: the statistics and z - m keep float32's accuracy.  No weight, no bias."""
    from magnet_amd.layer.norm import complex_group_norm
    x = _features(3000, 20, seed=8) + 1e4
    one, zero = torch.ones(20, dtype=torch.float64), torch.zeros(20, dtype=torch.float64)
    g = torch.randn(3000, 2, 20, generator=_gen(1))
    out, dx, _, _, tol_out, tol_dx, _, _ = _norm_reference(x, 4, one, zero, [3000], 1e-5, False, g)
    xd = x.to(DEV).requires_grad_()
    y = complex_group_norm(xd, 4)
    y.backward(g.to(DEV))
    # as above; mean |z|^2 - |m|^2 in 64 bits: 2^-53 * (10^4)^2 of the variance at worst, 0.2 u
    _close(y.detach(), out, 9 * U * tol_out + 1e-300, 'result')
    _close(xd.grad, dx, 22 * U * tol_dx + 1e-300, 'dx')


def test_group_norm_very_far_from_zero():
    """A mean 10^6 deviations from 0 (16 steps of float32 to a deviation): the deviations' own accuracy, and behind rows that are NaN."""
    from magnet_amd.layer.norm import complex_group_norm
    n, f, groups = 3000, 20, 4
    x = torch.randn(n, 2, f, generator=_gen(8)) + 1e6
    one, zero = torch.ones(f, dtype=torch.float64), torch.zeros(f, dtype=torch.float64)
    g = torch.randn(n, 2, f, generator=_gen(1))
    g[2500:] = 0
    sizes = [1000, 1500]
    out, dx, _, _, tol_out, tol_dx, _, _ = _norm_reference(x, groups, one, zero, sizes, 1e-5, False, g)
    xd = x.to(DEV)
    xd[2500:] = float('nan')
    xd.requires_grad_()
    y = complex_group_norm(xd, groups, graph_ptr=torch.tensor([0, 1000, 2500], device=DEV))
    y.backward(g.to(DEV))
    # as above; the mean is kept to 2^-48 of itself, the reference's own sums of 15000 values to less than 2^-47 (14 levels of
    # additions); the deviation of both parts together is sqrt(2): 2^-46 * 10^6 covers both
    far = 2.0 ** -46 * 1e6
    _close(y.detach(), out, 9 * U * tol_out + far, 'result')
    _close(xd.grad, dx, 22 * U * tol_dx + 4 * far * float(tol_dx.max()), 'dx')
    assert not bool(y[2500:].any()) and not bool(xd.grad[2500:].any())


def test_group_norm_gradient_against_differences():
    from magnet_amd.layer.norm import complex_group_norm
    x, w, b = _features(37, 12, seed=2), 0.5 + torch.rand(12, generator=_gen(3)), torch.randn(12, generator=_gen(4))
    g = torch.randn(37, 2, 12, generator=_gen(6)).double()
    ts = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    loss = lambda *t: float((complex_group_norm(t[0], 3, t[1], t[2]).detach().double().cpu() * g).sum())
    complex_group_norm(ts[0], 3, ts[1], ts[2]).backward(g.float().to(DEV))
    for i, t in enumerate(ts):
        d = torch.randn(t.shape, generator=_gen(10 + i)).to(DEV)
        h = 2.0 ** -7
        moved = [[s.detach() + (sign * h * d if j == i else 0) for j, s in enumerate(ts)] for sign in (1, -1)]
        numeric = (loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        analytic = float((t.grad.double() * d.double()).sum())
        # second-order differences: h^2 times a third derivative of order |d|^3 / sd^2, and u / h from the results' roundings
        assert abs(numeric - analytic) <= 2e-3 * float((t.grad.abs() * d.abs()).sum()) + 1e-6


def test_group_norm_strided_input_gradient_and_block_output():
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.sparse_magnet import _block_of
    block = _features(90, 3 * 16, seed=12).to(DEV).view(90, 2, 3, 16)
    plain = complex_group_norm(block[:, :, 1, :].contiguous(), 4, relu=True)
    y = complex_group_norm(block[:, :, 1, :], 4, relu=True, next_terms=3)
    assert torch.equal(plain, y) and tuple(_block_of(y, 3).shape) == (90, 2, 3, 16)
    odd = block.view(90, 2, 48)[:, :, 1:17]                        # off 16 bytes: the scalar path
    _close(complex_group_norm(odd, 4), complex_group_norm(odd.contiguous(), 4).double().cpu(), torch.full((1,), 1e-5, dtype=torch.float64), 'scalar path')
    grads = []
    for kind in range(4):
        x = block[:, :, 1, :].detach().clone().requires_grad_()
        y = complex_group_norm(x, 4)
        base = torch.randn(1, 1, 16, generator=_gen(1)).to(DEV)
        g = base.expand(90, 2, 16)
        if kind == 1:
            g = g.contiguous()
        elif kind == 2:
            g = g.transpose(0, 1).contiguous().transpose(0, 1)
        elif kind == 3:
            g = g.transpose(1, 2).contiguous().transpose(1, 2)
        y.backward(g)
        grads.append(x.grad)
    assert all(torch.equal(grads[0], t) for t in grads[1:])
    x = block[:, :, 1, :].detach().clone().requires_grad_()
    complex_group_norm(x, 4).sum().backward()                      # a gradient that is one value expanded
    assert float(x.grad.abs().max()) <= 1e-5


def test_group_norm_values_that_are_not_finite_stay_in_their_group():
    from magnet_amd.layer.norm import complex_group_norm
    x = _features(60, 8, seed=4)
    ptr = torch.tensor([0, 20, 60], dtype=torch.int32, device=DEV)
    clean = complex_group_norm(x.to(DEV), 2, graph_ptr=ptr, relu=True)
    x[3, 1, 5] = float('inf')
    got = complex_group_norm(x.to(DEV), 2, graph_ptr=ptr, relu=True)
    assert bool(torch.isnan(got[:20, :, 4:]).all())
    assert torch.equal(got[:20, :, :4], clean[:20, :, :4]) and torch.equal(got[20:], clean[20:])


def test_group_norm_refusals():
    from magnet_amd import MagnetHipError
    from magnet_amd.layer.norm import complex_group_norm
    x = torch.zeros(6, 2, 8, device=DEV)
    for call in (lambda: complex_group_norm(x, 3), lambda: complex_group_norm(x, 0), lambda: complex_group_norm(x.double(), 2),
                 lambda: complex_group_norm(x, 2, torch.ones(7, device=DEV)), lambda: complex_group_norm(x, 2, torch.ones(8)),
                 lambda: complex_group_norm(x, 2, None, torch.ones(8, device=DEV).double()),
                 lambda: complex_group_norm(x, 2, graph_ptr=torch.tensor([0, 6])),
                 lambda: complex_group_norm(x, 2, graph_ptr=torch.tensor([0], device=DEV)),
                 lambda: complex_group_norm(x, 2, graph_ptr=torch.zeros((2, 2), dtype=torch.int32, device=DEV))):
        with pytest.raises(MagnetHipError):
            call()
    empty = torch.zeros(0, 2, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = complex_group_norm(empty, 2, w)
    y.sum().backward()
    assert y.shape == (0, 2, 8) and not bool(w.grad.any())
    assert complex_group_norm(empty.detach(), 2, graph_ptr=torch.tensor([0, 0], device=DEV)).shape == (0, 2, 8)


# ---------------------------------------------------------------------------------------------
# class scores
# ---------------------------------------------------------------------------------------------
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _score_case(rows, classes, layout, type_, seed):
    s = (3 * torch.randn(rows, classes, generator=_gen(seed))).to(TYPES[type_])
    lab = torch.randint(0, classes, (rows,), generator=_gen(seed + 1))
    lab[torch.rand(rows, generator=_gen(seed + 2)) < 0.3] = -100
    if rows:
        lab[0] = classes - 1
    return s, lab


def _given(s, lab, layout):
    """[rows, classes] as the operators take it: [M, C], [1, C, N], [2, C, N / 2], or a strided view of something wider."""
    if layout == 'row':
        return s.to(DEV), lab.to(DEV)
    if layout == 'class':
        return s.t().contiguous().unsqueeze(0).to(DEV), lab.unsqueeze(0).to(DEV)
    if layout == 'batch':
        n = s.size(0) // 2
        return s.view(2, n, -1).transpose(1, 2).contiguous().to(DEV), lab.view(2, n).to(DEV)
    wide = torch.zeros(s.size(0), 2 * s.size(1) + 1, dtype=s.dtype, device=DEV)
    wide[:, 1::2] = s.to(DEV)
    return wide[:, 1::2], lab.to(DEV)


def _rowwise(t, layout):
    """Anything of the scores' layout back to [rows, ...] on the host."""
    t = t.detach().cpu()
    if layout == 'class':
        return t[0].t() if t.dim() == 3 else t[0]
    if layout == 'batch':
        return t.transpose(1, 2).reshape(-1, t.size(1)) if t.dim() == 3 else t.reshape(-1)
    return t


SCORE_CASES = [(1, 1, 'row'), (1, 2, 'class'), (2, 3, 'batch'), (63, 5, 'class'), (64, 5, 'row'), (65, 8, 'class'), (130, 9, 'row'), (100, 17, 'class'),
               (1000, 5, 'strided'), (2500, 5, 'class'), (2500, 3, 'row'), (300, 64, 'batch'), (77, 65, 'row'), (40, 349, 'row'), (40, 349, 'class'),
               (3, 513, 'row'), (1, 1500, 'row'), (5, 4097, 'class'), (5, 4097, 'row'), (9, 1030, 'strided'), (140000, 20, 'class')]


@pytest.mark.parametrize('type_', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows,classes,layout', SCORE_CASES)
def test_class_logprobs_and_their_gradients(rows, classes, layout, type_):
    from magnet_amd.layer.scores import class_logprobs
    top = min(classes, (rows + classes) % 7 + (16 if classes == 349 else 0), 16)
    s, lab = _score_case(rows, classes, layout, type_, rows + classes)
    x = s.double()
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    h = -(p * lp).sum(1)
    want = torch.where(lab >= 0, lp.gather(1, lab.clamp(min=0).unsqueeze(1)).squeeze(1), 0.0)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    sd, labd = _given(s, lab, layout)
    sd.requires_grad_()
    r = class_logprobs(sd, labd, top=top)
    assert r.logprob.shape == r.entropy.shape == labd.shape and r.logprob.dtype == torch.float32
    # e^x to 2 u, a sum of up to `classes` terms, log to 2 u, the differences u each of what they subtract
    depth = (classes + 16) * U
    spread = (x.amax(1) - x.amin(1)) + 1
    _close(_rowwise(r.logprob, layout), want, depth + 4 * U * (want.abs() + spread), 'logprob')
    _close(_rowwise(r.entropy, layout), h, (2 * depth + 8 * U) * (1 + h + (p * (x.amax(1, keepdim=True) - x)).sum(1)), 'entropy')
    if top:
        assert torch.equal(_rowwise(r.top_index, layout), order)
        best = lp.gather(1, order)
        _close(_rowwise(r.top_logprob, layout), best, depth + 4 * U * (best.abs() + spread.unsqueeze(1)), 'top')
    gl, gh, gt = (torch.randn(v, generator=_gen(k)) for k, v in ((1, (rows,)), (2, (rows,)), (3, (rows, top))))
    shaped = lambda t: _given(t, lab, 'row' if layout == 'strided' else layout)[0] if t.dim() == 2 else _given(s, t, layout)[1]
    torch.autograd.backward([r.logprob, r.entropy] + ([r.top_logprob] if top else []), [shaped(gl), shaped(gh)] + ([shaped(gt)] if top else []))
    one = torch.zeros_like(x)
    use = lab >= 0
    a = torch.where(use, gl.double(), 0.0)
    one[use] = one[use].scatter(1, lab[use].unsqueeze(1), a[use].unsqueeze(1))
    for t in range(top):
        one.scatter_add_(1, order[:, t:t + 1], gt[:, t:t + 1].double())
    total = a + gt.double().sum(1)
    d = one - p * total.unsqueeze(1) - p * (lp + h.unsqueeze(1)) * gh.double().unsqueeze(1)
    size = one.abs() + p * (a.abs() + gt.double().abs().sum(1)).unsqueeze(1) + p * (lp.abs() + h.unsqueeze(1) + 1) * gh.double().abs().unsqueeze(1)
    # p to the accuracy of its logarithm, 24 operations at most (16 of them the alternatives), one rounding to the type
    tol = (depth + 4 * U * (spread.unsqueeze(1) + lp.abs()) + 24 * U) * 2 * size + torch.finfo(TYPES[type_]).eps / 2 * d.abs()
    if type_ == 'f16':
        tol = tol + 2.0 ** -25                                     # half a step of its subnormal numbers
    assert sd.grad.dtype == sd.dtype
    _close(_rowwise(sd.grad, layout), d, tol + 1e-38, 'gradient')


@pytest.mark.parametrize('type_', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows,classes,layout', SCORE_CASES)
def test_class_nll_and_its_gradient(rows, classes, layout, type_):
    from magnet_amd.layer.scores import class_nll
    s, lab = _score_case(rows, classes, layout, type_, rows + 3 * classes)
    x = s.double()
    lp = torch.log_softmax(x, 1)
    use = lab >= 0
    count = int(use.sum())
    per_row = -lp[use].gather(1, lab[use].unsqueeze(1)).squeeze(1)
    sd, labd = _given(s, lab, layout)
    sd.requires_grad_()
    loss, acc = class_nll(sd, labd)
    (3.0 * loss).backward()
    spread = float((x.amax(1) - x.amin(1)).max()) + 1
    tol = (classes + 16) * U + 4 * U * (float(per_row.abs().max()) + spread)     # of every row, so of their mean; one rounding of it
    loss, acc = loss.detach(), acc.detach()
    assert abs(float(loss) - float(per_row.mean())) <= tol + U * float(per_row.mean())
    first = torch.sort(x, dim=1, descending=True, stable=True)[1][:, 0]
    assert float(acc) == float(torch.tensor(int((first[use] == lab[use]).sum()) / count, dtype=torch.float32))
    d = torch.zeros_like(x)
    d[use] = lp[use].exp()
    d[use] = d[use].scatter_add(1, lab[use].unsqueeze(1), torch.full((count, 1), -1.0, dtype=torch.float64))
    d *= 3.0 / count
    rel = (classes + 24) * U + 4 * U * (spread + lp.abs())
    bound = 2 * rel * 3.0 / count + torch.finfo(TYPES[type_]).eps / 2 * d.abs() + (2.0 ** -25 if type_ == 'f16' else 1e-38)
    _close(_rowwise(sd.grad, layout), d, bound, 'gradient')
    assert not bool(_rowwise(sd.grad, layout)[~use].any())
    a, b = class_nll(sd.detach(), labd)                            # no gradient wanted: the same numbers
    assert float(a) == float(loss) and float(b) == float(acc)


@pytest.mark.parametrize('type_', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('batch,inner,classes,gap,special', [(1, 65536, 2, 0, False), (1, 65537, 3, 0, True), (1, 70002, 5, 1, True), (3, 30003, 8, 0, True),
                                                             (250, 263, 7, 2, False), (1, 300003, 4, 3, True), (2, 40001, 6, 0, False),
                                                             (1, 65535, 5, 0, True)])
def test_class_nll_of_many_rows(batch, inner, classes, gap, special, type_):
    """Class-major scores of few classes: rows that do not divide by 4, `gap` values between the classes' rows (so that every class
    starts at another alignment), ignored rows, rows without a distribution."""
    from magnet_amd.layer.scores import class_nll
    g = _gen(inner + classes)
    wide = (2 * torch.randn(batch, classes, inner + gap, generator=g)).to(TYPES[type_]).to(DEV)
    lab = torch.randint(-1, classes, (batch, inner), generator=g)
    lab[lab < 0] = -100
    s = wide[:, :, :inner]
    rows = s.permute(0, 2, 1).reshape(-1, classes).double().cpu()
    flat = lab.reshape(-1)
    use = flat >= 0
    if special:                                                    # rows that nothing counts may hold anything
        odd = torch.nonzero(~use)[:4, 0]
        for at, v in zip(odd.tolist(), (float('nan'), float('inf'), -float('inf'), 0.0)):
            s[at // inner, :, at % inner] = v
        masked = torch.nonzero(use)[:3, 0]
        for at in masked.tolist():                                 # a class without probability that is not the label
            c = (int(flat[at]) + 1) % classes
            s[at // inner, c, at % inner] = -float('inf')
            rows[at, c] = -float('inf')
    sd = s.detach().requires_grad_()
    loss, acc = class_nll(sd, lab.to(DEV))
    (3.0 * loss).backward()
    lp = torch.log_softmax(rows, 1)
    count = int(use.sum())
    per_row = -lp[use].gather(1, flat[use].unsqueeze(1)).squeeze(1)
    finite = torch.where(torch.isfinite(rows), rows, torch.zeros_like(rows))
    spread = float((finite.amax(1) - finite.amin(1)).max()) + 1
    loss, acc = loss.detach(), acc.detach()
    # as for the other layouts
    tol = (classes + 16) * U + 4 * U * (float(per_row.abs().max()) + spread)
    assert abs(float(loss) - float(per_row.mean())) <= tol + U * float(per_row.mean())
    first = torch.sort(rows, dim=1, descending=True, stable=True)[1][:, 0]
    assert float(acc) == float(torch.tensor(int((first[use] == flat[use]).sum()) / count, dtype=torch.float32))
    d = torch.zeros_like(rows)
    d[use] = lp[use].exp()
    d[use] = d[use].scatter_add(1, flat[use].unsqueeze(1), torch.full((count, 1), -1.0, dtype=torch.float64))
    d *= 3.0 / count
    rel = (classes + 24) * U + 4 * U * (spread + lp.abs().clamp(max=1e3))
    bound = 2 * rel * 3.0 / count + torch.finfo(TYPES[type_]).eps / 2 * d.abs() + (2.0 ** -25 if type_ == 'f16' else 1e-38)
    got = sd.grad.permute(0, 2, 1).reshape(-1, classes).cpu()
    _close(got, d, bound, 'gradient')
    assert not bool(got[~use].any())
    a, b = class_nll(sd.detach(), lab.to(DEV))
    assert float(a) == float(loss) and float(b) == float(acc)
    # a counted row without a distribution, a label out of range: NaN where they are, and nowhere else in the gradient
    at = int(torch.nonzero(use)[5, 0])
    for kind in ('masked', 'label'):
        s2, lab2 = s.detach().clone(), lab.clone()
        if kind == 'masked':
            s2[at // inner, :, at % inner] = -float('inf')
        else:
            lab2[at // inner, at % inner] = classes
        s2.requires_grad_()
        bad = class_nll(s2, lab2.to(DEV))[0]
        bad.backward()
        got = torch.isnan(s2.grad.permute(0, 2, 1).reshape(-1, classes)).cpu()
        assert bool(torch.isnan(bad)) and bool(got[at].all()) and int(got.sum()) == classes


@pytest.mark.parametrize('layout,classes', [('row', 5), ('class', 5), ('row', 40), ('class', 40), ('row', 1100)])
def test_scores_with_masks_and_values_that_are_not_finite(layout, classes):
    from magnet_amd.layer.scores import class_logprobs, class_nll
    s = 2 * torch.randn(9, classes, generator=_gen(classes))
    low = torch.finfo(torch.float32).min
    s[1, ::2] = -float('inf')                                      # masked classes
    s[2] = -float('inf')                                           # nothing left
    s[3] = low                                                     # masked with the type's lowest value: uniform
    s[4, 1:] = low
    s[4, 0] = 3e38                                                 # their difference is not a float
    s[5, 3] = float('nan')
    s[6, 2] = float('inf')
    s[7, :] = 0.0
    s[7, classes - 1] = -0.0                                       # a tie
    s[8] = -float('inf')
    s[8, 2] = -7.0                                                 # one class left
    lab = torch.tensor([0, 1, 0, 1, 0, 2, 1, 0, 2])
    sd, labd = _given(s, lab, layout)
    sd.requires_grad_()
    top = min(classes, 5)
    r = class_logprobs(sd, labd, top=top)
    lp = torch.log_softmax(s.double(), 1)
    got_lp, got_h = _rowwise(r.logprob, layout), _rowwise(r.entropy, layout)
    want = lp.gather(1, lab.unsqueeze(1)).squeeze(1)
    assert bool((torch.isnan(got_lp) == torch.isnan(want)).all())
    fine = torch.isfinite(want)
    _close(got_lp[fine], want[fine], 64 * U * (1 + want[fine].abs()) + classes * U, 'logprob')
    h = torch.special.entr(lp.exp()).sum(1)
    assert bool((torch.isnan(got_h) == torch.isnan(h)).all())
    ok = ~torch.isnan(h)
    _close(got_h[ok], h[ok], (64 + 2 * classes) * U * (1 + h[ok]), 'entropy')
    idx = _rowwise(r.top_index, layout)
    for i in (0, 1, 3, 4, 7, 8):
        clean = torch.sort(s[i].double() + 0.0, descending=True, stable=True)[1][:top]
        assert torch.equal(idx[i], clean), i
    assert idx[5, 0] == 3 and idx[6, 0] == 2 and torch.equal(idx[2], torch.arange(top))
    # gradients: rows no gradient reaches stay clean whatever they hold; a masked class gets none
    pick = torch.tensor([1., 1, 0, 1, 1, 0, 0, 1, 1])
    g = _given(s, pick, layout)[1]
    torch.autograd.backward([r.logprob, r.entropy], [g, g])
    d = _rowwise(sd.grad, layout)
    assert not bool(d[[2, 5, 6]].any()) and not bool(d[1, ::2].any()) and bool(torch.isfinite(d).all())
    # the loss of the rows that can have one; ignored rows may hold anything
    lab2 = torch.where(pick > 0, lab, torch.full_like(lab, -100))
    sd2, labd2 = _given(s, lab2, layout)
    sd2.requires_grad_()
    loss, _ = class_nll(sd2, labd2)
    loss.backward()
    loss = loss.detach()
    rows = pick > 0
    assert float(loss) == pytest.approx(float(-want[rows].mean()), rel=1e-5)
    d = _rowwise(sd2.grad, layout)
    assert bool(torch.isfinite(d).all()) and not bool(d[~rows].any())
    # a label out of range is NaN, and nothing is read out of range
    for bad in (classes, -1, 2 ** 40):
        lab3 = lab.clone()
        lab3[0] = bad
        sd3, labd3 = _given(s, lab3, layout)
        got = _rowwise(class_logprobs(sd3, labd3).logprob, layout)
        assert bool(torch.isnan(got[0])) and bool(torch.isfinite(got[8]))
        assert bool(torch.isnan(class_nll(sd3[:1] if layout == 'row' else sd3[:, :, :1], labd3[:1] if layout == 'row' else labd3[:, :1])[0]))


@pytest.mark.parametrize('type_', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('layout,classes', [('row', 5), ('class', 7), ('row', 64), ('row', 349), ('class', 40), ('row', 1536), ('row', 1600)])
def test_order_of_the_alternatives(layout, classes, type_):
    """Ties to the lower class, -0 equal to 0, NaN of either sign before all, masked classes last and in order."""
    from magnet_amd.layer.scores import class_logprobs, class_nll
    s = torch.randint(-3, 4, (8, classes), generator=_gen(classes)).to(TYPES[type_])         # ties everywhere
    s[1] = s[1] * 0.0                                              # zeros of both signs
    s[2, 1:] = -float('inf')
    s[3] = -float('inf')
    nan = torch.tensor([float('nan')]).to(TYPES[type_])
    s[4, 2], s[4, 4] = nan[0], -nan[0]
    s[5, classes - 1] = float('inf')
    tiny = torch.finfo(TYPES[type_]).smallest_normal
    s[6] = torch.randint(-2, 3, (classes,), generator=_gen(1)).to(TYPES[type_]) * tiny
    s[7] = torch.randn(classes, generator=_gen(2)).to(TYPES[type_])
    lab = torch.zeros(8, dtype=torch.int64)
    top = min(16, classes)
    sd, labd = _given(s, lab, layout)
    r = class_logprobs(sd, labd, top=top)
    inf = float('inf')
    order = torch.sort(torch.nan_to_num(s.double() + 0.0, nan=inf, posinf=inf, neginf=-inf), dim=1, descending=True, stable=True)[1][:, :top]
    got = _rowwise(r.top_index, layout)
    assert torch.equal(got, order)
    value, lp = _rowwise(r.top_logprob, layout).double(), torch.log_softmax(s.double(), 1).gather(1, order)
    for i in (0, 1, 2, 6, 7):
        fine = torch.isfinite(lp[i])
        assert torch.equal(torch.isfinite(value[i]), fine)
        assert float((value[i] - lp[i])[fine].abs().max()) <= (classes + 64) * U * 16        # log p below 16, as in the other tests
    # the best class of the loss is the first of them
    for i in (0, 1, 6, 7):
        one = _given(s[i:i + 1], order[i:i + 1, 0], layout)
        assert float(class_nll(*one)[1]) == 1.0


@pytest.mark.parametrize('layout,classes', [('row', 3), ('row', 16), ('row', 80), ('class', 5), ('row', 1100)])
def test_gradient_of_a_row_without_a_distribution(layout, classes):
    """A row of -inf alone has a log probability and an entropy of NaN, and so has its gradient; its neighbours keep theirs."""
    from magnet_amd.layer.scores import class_logprobs, class_nll
    s = torch.randn(6, classes, generator=_gen(classes))
    s[2] = -float('inf')
    lab = torch.tensor([0, 1, 1, 2, 0, 1])
    sd, labd = _given(s, lab, layout)
    for loss in (lambda t: class_nll(t, labd)[0], lambda t: class_logprobs(t, labd).logprob.sum(), lambda t: class_logprobs(t).entropy.sum()):
        t = sd.clone().requires_grad_()
        loss(t).backward()
        d = _rowwise(t.grad, layout)
        assert bool(torch.isnan(d[2]).all()) and bool(torch.isfinite(d[[0, 1, 3, 4, 5]]).all())


def test_scores_without_rows_labels_or_gradients():
    from magnet_amd import MagnetHipError
    from magnet_amd.layer.scores import class_logprobs, class_nll
    r = class_logprobs(torch.zeros(0, 4, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), top=2)
    assert r.logprob.shape == (0,) and r.top_index.shape == (0, 2)
    loss, acc = class_nll(torch.zeros(0, 4, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV))
    assert bool(torch.isnan(loss)) and bool(torch.isnan(acc))
    s = torch.randn(7, 4, device=DEV, requires_grad=True)
    r = class_logprobs(s)
    assert r.logprob is None and r.top_logprob.shape == (7, 0)
    r.entropy.sum().backward()                                     # one value expanded over the rows
    first = s.grad.clone()
    s.grad = None
    class_logprobs(s).entropy.backward(torch.ones(7, device=DEV))
    assert torch.equal(first, s.grad)
    loss, _ = class_nll(s, torch.full((7,), -100, device=DEV))
    assert bool(torch.isnan(loss))                                 # nothing to average, as torch's loss has it
    lab = torch.zeros(7, dtype=torch.int64, device=DEV)
    for call in (lambda: class_nll(s.double(), lab), lambda: class_nll(s, lab.int()), lambda: class_nll(s, lab.cpu()),
                 lambda: class_logprobs(torch.zeros(3, 0, device=DEV)), lambda: class_nll(torch.zeros(3, 2, 2, 2, device=DEV), lab)):
        with pytest.raises(MagnetHipError):
            call()
    wide = torch.randn(1, 4, 1, device=DEV).expand(1, 4, 50).requires_grad_()        # one node's scores for all
    class_nll(wide, torch.zeros((1, 50), dtype=torch.int64, device=DEV))[0].backward()
    assert float(wide.grad.sum().abs()) <= 1e-6


def test_nll_gradient_against_differences():
    from magnet_amd.layer.scores import class_logprobs, class_nll
    s = torch.randn(1, 6, 300, generator=_gen(1)).to(DEV).requires_grad_()
    lab = torch.randint(0, 6, (1, 300), generator=_gen(2)).to(DEV)
    f = lambda t: class_nll(t, lab)[0] - 0.3 * class_logprobs(t).entropy.mean()
    f(s).backward()
    d = torch.randn(1, 6, 300, generator=_gen(3)).to(DEV)
    h = 2.0 ** -6
    numeric = (float(f(s.detach() + h * d)) - float(f(s.detach() - h * d))) / (2 * h)
    analytic = float((s.grad.double() * d.double()).sum())
    # h^2 / 6 of a third derivative of order |d|^3, and 4 u of the losses over 2 h
    assert abs(numeric - analytic) <= h * h * float((s.grad.abs() * d.abs() ** 3).sum()) + 64 * U / h


# ---------------------------------------------------------------------------------------------
# together, as a training step uses them
# ---------------------------------------------------------------------------------------------
def _graph(n, e, q=0.15, seed=3):
    from magnet_amd.laplacian import build_magnetic_laplacian, powerlaw_edges
    src, dst = powerlaw_edges(n, e, seed, device=DEV)
    return build_magnetic_laplacian(src, dst, n, q=q)


def _net(cls, lap, cin, seed=0, **kw):
    from magnet_amd.utils.hermitian import ChebBasis
    torch.manual_seed(seed)
    net = cls(cin, ChebBasis(lap, 2), None, K=2, activation=True, **kw).to(DEV)
    g = _gen(seed)
    for name, p in net.named_parameters():
        if p.dim() == 1 and 'Chebs' in name:                       # norms off their initial ones and zeros
            p.data += 0.3 * torch.randn(p.shape, generator=g).to(DEV)
    return net


def _plain_trunk(net, lap, x, ptr):
    """The network's convolutions, norms and gates in 64 bits on the host, for autograd: complex [N, C] in and out."""
    from magnet_amd.layer.norm import ComplexGroupNorm
    from magnet_amd.layer.sparse_magnet import ChebConv
    L = torch.from_numpy(lap.to_scipy().toarray().astype(np.complex128))
    params = {k: v.detach().double().cpu().requires_grad_() for k, v in net.named_parameters()}
    z = x
    for i, m in enumerate(net.Chebs):
        name = 'Chebs.%d.' % i
        if isinstance(m, ChebConv):
            t = [z, L @ z]
            while len(t) < m.weight.size(0):
                t.append(2 * (L @ t[-1]) - t[-2])
            z = sum(a @ params[name + 'weight'][k].to(torch.complex128) for k, a in enumerate(t))
            z = z + torch.complex(params[name + 'bias'], params[name + 'bias'])
        elif isinstance(m, ComplexGroupNorm):
            rows = []
            for a, b in zip(ptr[:-1], ptr[1:]):
                v = z[a:b].view(b - a, m.num_groups, -1)
                mean = v.mean((0, 2), keepdim=True)
                var = ((v - mean).real ** 2 + (v - mean).imag ** 2).mean((0, 2), keepdim=True)
                rows.append(((v - mean) / torch.sqrt(var + m.eps)).view(b - a, -1))
            z = torch.cat(rows) * params[name + 'weight'] + torch.complex(params[name + 'bias'], params[name + 'bias'])
        else:
            z = z * (z.real >= 0)
    return z, params


@pytest.mark.parametrize('layer,graphs', [(2, (150, 250)), (3, (400,))])
def test_network_with_norms_against_64_bits(layer, graphs):
    """Scores, loss and every gradient of conv -> norm -> gate ... -> scores -> loss."""
    from magnet_amd.layer.scores import class_nll
    from magnet_amd.layer.sparse_magnet import ChebNet
    n, cin = sum(graphs), 6
    lap = _graph(n, 5 * n)
    ptr = np.concatenate([[0], np.cumsum(graphs)])
    net = _net(ChebNet, lap, cin, num_filter=12, label_dim=4, layer=layer, norm_groups=3,
               graph_ptr=torch.tensor(ptr, dtype=torch.int32, device=DEV))
    assert 'graph_ptr' not in net.state_dict()
    real, imag = torch.randn(n, cin, generator=_gen(1)), torch.randn(n, cin, generator=_gen(2))
    lab = torch.randint(0, 4, (1, n), generator=_gen(3))
    loss, _ = class_nll(net.scores(net.trunk(real.to(DEV), imag.to(DEV))), lab.to(DEV))
    loss.backward()
    loss = loss.detach()
    z, params = _plain_trunk(net, lap, torch.complex(real.double(), imag.double()), ptr)
    feats = torch.cat((z.real, z.imag), 1)
    scores = feats @ params['Conv.weight'].squeeze(-1).t() + params['Conv.bias']
    want = torch.nn.functional.cross_entropy(scores, lab[0])
    want.backward()
    # the framework's bar for float32 forward and backward results, 1e-5 of a tensor's largest value; a gate on the border of 0
    # may open one value of float32's accuracy on the other side
    assert abs(float(loss) - want.item()) <= 1e-5 * abs(want.item())
    for k, p in net.named_parameters():
        ref = params[k].grad
        assert float((p.grad.double().cpu() - ref).abs().max()) <= 2e-5 * float(ref.abs().max()) + 1e-9, k


@pytest.mark.parametrize('filters,cin', [(12, 6), (8, 20)])
def test_network_with_checkpoints_in_8_bits(filters, cin):
    """cin 20 > 8 filters: the GEMM-first form keeps its input, the others their blocks of orders.  Forward and the gradient
    that reaches the input are those of 32 bits without norms; a weight gradient is off by what half a step of each kept value
    can do."""
    from magnet_amd.checkpoint import Checkpoint8
    from magnet_amd.layer.sparse_magnet import ChebNet, ChebConv, _as_packed, _cheb_terms
    n = 500
    lap = _graph(n, 2500)
    real, imag = torch.randn(n, cin, generator=_gen(1)).to(DEV), torch.randn(n, cin, generator=_gen(2)).to(DEV)
    outs, grads = [], []
    for bits in (32, 8):
        net = _net(ChebNet, lap, cin, num_filter=filters, label_dim=4, layer=2, checkpoint_bits=bits)
        r, i = real.clone().requires_grad_(), imag.clone().requires_grad_()
        out = net.trunk(r, i)
        out.backward(torch.randn(out.shape, generator=_gen(5)).to(DEV))
        outs.append(out.detach())
        grads.append([r.grad, i.grad] + [p.grad for k, p in net.named_parameters() if k.startswith('Chebs')])
    assert torch.equal(outs[0], outs[1])
    for a, b, name in zip(grads[0], grads[1], ['real', 'imag'] + [k for k, _ in net.named_parameters() if k.startswith('Chebs')]):
        if 'weight' not in name:
            assert torch.equal(a, b), name
        else:
            assert not torch.equal(a, b)
            # a value is off by at most 1 / 127.5 of the largest of its 32, which is below 4 of their root mean squares; with
            # signs that do not follow the gradient's the sum is off by that share of itself
            assert float((a - b).norm()) <= 4 / 127.5 * float(a.norm()), name
    # the weight gradient of one convolution is the gram of its checkpoint, to the bit
    conv = ChebConv(cin, filters, 2, net.Chebs[0].mul_L_real, None).to(DEV)
    conv.checkpoint_bits = 8
    x = _as_packed(real, imag)
    y = conv.forward_packed(x)
    g = torch.randn(y.shape, generator=_gen(6)).to(DEV)
    y.backward(g)
    if filters >= cin:
        want = Checkpoint8.store(_cheb_terms(lap, x, 3)).gram(g).view(3, cin, filters)
    else:
        want = Checkpoint8.store(x).gram(_cheb_terms(lap, g, 3)).view(cin, 3, filters).permute(1, 0, 2)
    assert torch.equal(conv.weight.grad, want)


def test_checkpoints_shrink_what_a_forward_keeps():
    from magnet_amd.layer.sparse_magnet import ChebNet
    n, f = 20000, 64
    lap = _graph(n, 60000)
    x = torch.randn(n, f, generator=_gen(1)).to(DEV)
    kept = {}
    for bits in (32, 8):
        net = _net(ChebNet, lap, f, num_filter=f, label_dim=4, layer=3, norm_groups=4, checkpoint_bits=bits)
        net(x, x)                                                  # plans and library handles
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = net.trunk(x, x)
        kept[bits] = torch.cuda.memory_allocated() - before - out.numel() * 4
        del out
    # kept per value of a block and of a norm's input: 4 bytes, or 1.03 and a byte for the gate of two values
    assert kept[8] < 0.36 * kept[32], kept


@pytest.mark.parametrize('dropout', [0.0])
def test_fused_loss_epochs_follow_the_plain_ones(dropout):
    from magnet_amd.layer.sparse_magnet import ChebNet, ChebNet_Edge
    from magnet_amd.train import NodeTargets, SharedForwardEpochs, link_epoch, node_epoch
    n = 600
    lap = _graph(n, 3000)
    x = torch.randn(n, 3, generator=_gen(1)).to(DEV)
    lab = torch.randint(0, 5, (1, n), generator=_gen(2)).to(DEV)
    train, val = torch.arange(0, 300, device=DEV), torch.arange(300, 450, device=DEV)
    pairs = torch.randint(0, n, (800, 2), generator=_gen(3)).to(DEV)
    y = torch.randint(0, 3, (800,), generator=_gen(4)).to(DEV)
    runs = []
    for fused, shared in ((False, False), (True, False), (True, True)):
        stats = []
        net = _net(ChebNet, lap, 3, num_filter=8, label_dim=5, layer=2, norm_groups=2, dropout=dropout)
        opt = torch.optim.Adam(net.parameters(), lr=1e-3)
        targets = (NodeTargets(lab, train), NodeTargets(lab, val)) if shared else (train, val)
        body = SharedForwardEpochs(net, opt, fused_loss=fused).node_epoch if shared else lambda *a: node_epoch(net, opt, *a, fused_loss=fused)
        for _ in range(4):
            stats += [float(v) for v in body(x, x, lab, *targets)]
        net = _net(ChebNet_Edge, lap, 3, num_filter=8, label_dim=3, layer=2, dropout=dropout)
        opt = torch.optim.Adam(net.parameters(), lr=1e-3)
        body = SharedForwardEpochs(net, opt, fused_loss=fused).link_epoch if shared else lambda *a: link_epoch(net, opt, *a, fused_loss=fused)
        for _ in range(4):
            stats += [float(v) for v in body(x, x, pairs[:500], y[:500], pairs[500:], y[500:])]
        runs.append(np.array(stats))
    # losses of the same steps to float32; an accuracy may move by a node whose two best classes are a rounding apart
    for r in runs[1:]:
        assert np.abs(r - runs[0]).max() <= 1e-2 and np.abs((r - runs[0])[0::2]).max() <= 1e-4


@pytest.mark.parametrize('kind', ['twice', 'mask', 'one'])
def test_fused_loss_of_index_tensors_counts_as_the_plain_one(kind):
    """An index tensor that names nodes more than once, a boolean mask, a single node."""
    from magnet_amd.layer.sparse_magnet import ChebNet
    from magnet_amd.train import node_epoch
    n = 300
    lap = _graph(n, 1500)
    x = torch.randn(n, 3, generator=_gen(1)).to(DEV)
    lab = torch.randint(0, 5, (1, n), generator=_gen(2)).to(DEV)
    index = {'twice': torch.tensor([3, 7, 3, 3, 250, 7], device=DEV), 'mask': torch.arange(n, device=DEV) % 3 == 0,
             'one': torch.tensor([11], device=DEV)}[kind]
    runs = []
    for fused in (False, True):
        net = _net(ChebNet, lap, 3, num_filter=8, label_dim=5, layer=2)
        opt = torch.optim.SGD(net.parameters(), lr=0.0)
        stats = [float(v) for v in node_epoch(net, opt, x, x, lab, index, index, fused_loss=fused)]
        runs.append((stats, [p.grad.clone() for p in net.parameters()]))
    # a loss is a mean of values below 8 with a few roundings each; gradients are products of as many
    assert np.abs(np.array(runs[0][0]) - np.array(runs[1][0])).max() <= 64 * U
    for a, b in zip(runs[0][1], runs[1][1]):
        assert float((a - b).abs().max()) <= 1e3 * U * float(a.abs().max()) + 1e-9


def test_training_epoch_as_hip_graphs_follows_the_eager_one():
    """Norms, 8-bit checkpoints and the fused loss under capture: every replay gives what an eager epoch gives, with the
    program's own work in between."""
    from magnet_amd.layer.sparse_magnet import ChebNet
    from magnet_amd.train import GraphedSharedEpochs, NodeTargets, SharedForwardEpochs
    n = 700
    lap = _graph(n, 3500)
    x = torch.randn(n, 4, generator=_gen(1)).to(DEV)
    lab = torch.randint(0, 5, (1, n), generator=_gen(2)).to(DEV)
    targets = [NodeTargets(lab, torch.arange(a, a + 200, device=DEV)) for a in (0, 300)]

    def make():
        net = _net(ChebNet, lap, 4, num_filter=16, label_dim=5, layer=2, norm_groups=4, checkpoint_bits=8)
        return net, torch.optim.Adam(net.parameters(), lr=1e-2, capturable=True)

    net, opt = make()
    shared = SharedForwardEpochs(net, opt, fused_loss=True)
    want = [[float(v) for v in shared.node_epoch(x, x, lab, *targets)] for _ in range(9)]
    del shared
    net, opt = make()
    graphed = GraphedSharedEpochs.for_nodes(net, opt, x, x, lab, *targets, warmup=3, fused_loss=True)
    for k in range(3, 9):
        got = [float(v) for v in graphed()]
        assert np.abs(np.array(got) - np.array(want[k])).max() <= 1e-4, (k, got, want[k])
        float(torch.randn(1000, device=DEV).sum())                 # the program's own work
        torch.cuda.synchronize()


def test_operators_replay_in_a_graph_and_run_on_other_streams():
    from magnet_amd.checkpoint import Checkpoint8
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.scores import class_logprobs, class_nll
    n, f = 3000, 24
    x, g = _features(n, f, seed=1).to(DEV), torch.randn(n, 2, 10, generator=_gen(2)).to(DEV)
    s = torch.randn(1, 7, n, generator=_gen(3)).to(DEV)
    lab = torch.randint(0, 7, (1, n), generator=_gen(4)).to(DEV)
    ptr = torch.tensor([0, 1000, 1000, 2900], dtype=torch.int32, device=DEV)

    def body():
        ck = Checkpoint8.store(x)
        r = class_logprobs(s, lab, top=3)
        return [ck.gram(g), ck.restore(), complex_group_norm(x, 3, graph_ptr=ptr, relu=True), *class_nll(s, lab), *r]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, body()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = body()
    for k in range(4):
        x.copy_(_features(n, f, seed=10 + k))
        s.copy_(torch.randn(1, 7, n, generator=_gen(20 + k)))
        graph.replay()
        torch.cuda.synchronize()
        want = body()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def test_drivers_take_the_new_arguments(tmp_path):
    from magnet_amd import Edge_sparseMagnet, sparse_Magnet
    root = str(tmp_path) + '/'
    common = ['--q', '0.1', '--K', '2', '-a', '--num_filter', '16', '--layer', '2', '--splits', '1', '--norm_groups', '4',
              '--checkpoint_bits', '8', '--fused_loss', '--report', '2', '--log_root', root, '--data_path', root]
    for extra in ([], ['--separate_forwards'], ['--hip_graph']):
        sparse_Magnet.run(['--dataset', 'syn/cyclic', '--p_q', '0.95', '--seed', '10', '--epochs', '4', '--new_setting'] + common + extra)
    Edge_sparseMagnet.run(['--dataset', 'syn/cyclic', '--task', '1', '--num_class_link', '2', '--epochs', '3'] + common)
    reports = sorted(tmp_path.rglob('report0.npz'))
    assert len(reports) >= 2
    for path in reports:
        r = np.load(path)
        assert set(r.files) == {'logprob', 'entropy', 'top_logprob', 'top_index'}
        assert (r['entropy'] >= -1e-6).all() and np.isfinite(r['logprob']).all() and r['top_index'].shape[1] == 2
        assert (np.diff(r['top_logprob'], axis=1) <= 0).all()


# ---------------------------------------------------------------------------------------------
# the C ABI with raw pointers, and calls at the edges of what the documentation allows
# ---------------------------------------------------------------------------------------------
def test_entry_points_with_raw_pointers():
    """Every entry point of the three operators as a caller without torch binds it, against the operators of the extension."""
    from magnet_amd import _lib
    from magnet_amd._lib import lib, ptr, stream_ptr, check
    from magnet_amd.checkpoint import Checkpoint8
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.scores import class_logprobs, class_nll
    n, f, k, s = 301, 20, 6, stream_ptr(torch.device(DEV, 0))
    x, g = _features(n, f, seed=1).to(DEV), torch.randn(n, 2, k, generator=_gen(2)).to(DEV)
    empty = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=DEV)
    ck = Checkpoint8.store(x)
    codes, scales, back, dw = torch.empty_like(ck.codes), torch.empty_like(ck.scales), torch.empty_like(x), empty(f, k)
    check(lib.mh_ckpt_store(ptr(x), 2 * f, f, n, f, ptr(codes), ptr(scales), s))
    check(lib.mh_ckpt_restore(ptr(codes), ptr(scales), n, f, ptr(back), 2 * f, f, s))
    size = lib.mh_ckpt_gram_workspace_bytes(n, f, k)
    ws = empty(size, dtype=torch.uint8)
    check(lib.mh_ckpt_gram(ptr(codes), ptr(scales), n, f, ptr(g), 2 * k, k, k, ptr(dw), ptr(ws), size, s))
    assert torch.equal(codes, ck.codes) and torch.equal(scales, ck.scales) and torch.equal(back, ck.restore()) and torch.equal(dw, ck.gram(g))
    w, b = (torch.rand(f, generator=_gen(i)).to(DEV) + 0.5 for i in (3, 4))
    go = torch.randn(n, 2, f, generator=_gen(5)).to(DEV)
    graphs = torch.tensor([0, 100, 290], dtype=torch.int32, device=DEV)
    size = lib.mh_group_norm_workspace_bytes(n, 2, f, 4)
    ws = empty(size, dtype=torch.uint8)
    for held in (False, True):
        xr, wr, br = (t.clone().requires_grad_() for t in (x, w, b))
        want = complex_group_norm(xr, 4, wr, br, graph_ptr=graphs, relu=True, checkpoint_bits=8 if held else 32)
        want.backward(go)
        y, mask, stats, dx, dgamma, dbeta = torch.empty_like(x), empty(n, f, dtype=torch.uint8), empty(2, 4, 5), torch.empty_like(x), empty(f), empty(f)
        check(lib.mh_group_norm(ptr(x), 2 * f, f, n, f, 4, ptr(graphs), 2, 1e-5, ptr(w), ptr(b), 1, ptr(y), 2 * f, f, ptr(mask),
                                ptr(codes) if held else None, ptr(scales) if held else None, ptr(stats), ptr(ws), size, s))
        check(lib.mh_group_norm_bwd(None if held else ptr(x), 2 * f, f, ptr(codes) if held else None, ptr(scales) if held else None, ptr(mask),
                                    n, f, 4, ptr(graphs), 2, ptr(stats), ptr(w), ptr(b), 1, ptr(go), 2 * f, f, ptr(dx), 2 * f, f, ptr(dgamma),
                                    ptr(dbeta), ptr(ws), size, s))
        assert torch.equal(y, want) and torch.equal(dx, xr.grad) and torch.equal(dgamma, wr.grad) and torch.equal(dbeta, br.grad)
        check(lib.mh_group_norm_bwd(None if held else ptr(x), 2 * f, f, ptr(codes) if held else None, ptr(scales) if held else None, ptr(mask),
                                    n, f, 4, ptr(graphs), 2, ptr(stats), ptr(w), ptr(b), 1, ptr(go), 2 * f, f, None, 0, 0, ptr(dgamma), None,
                                    ptr(ws), size, s))               # some gradients not wanted
        assert torch.equal(dgamma, wr.grad)
    c = 7
    sc = torch.randn(n, c, generator=_gen(6)).to(DEV).requires_grad_()
    lab = torch.randint(0, c, (n,), generator=_gen(7)).to(DEV)
    r = class_logprobs(sc, lab, top=3)
    gl, gh, gt = torch.randn(n, device=DEV), torch.randn(n, device=DEV), torch.randn(n, 3, device=DEV)
    torch.autograd.backward([r.logprob, r.entropy, r.top_logprob], [gl, gh, gt])
    lp, ent, stat, tl, ti, d = empty(n), empty(n), empty(n, 2), empty(n, 3), empty(n, 3, dtype=torch.int64), empty(n, c)
    check(lib.mh_class_logprobs(ptr(sc), 0, 1, n, c, 0, 1, c, ptr(lab), -100, ptr(lp), ptr(ent), ptr(stat), 3, ptr(tl), ptr(ti), 0, 1, 3, s))
    check(lib.mh_class_logprobs_bwd(ptr(sc), 0, 1, n, c, 0, 1, c, ptr(lab), -100, ptr(stat), ptr(ent), ptr(gl), 1, ptr(gh), 1, 3, ptr(gt), ptr(ti),
                                    0, 1, 3, ptr(d), 0, 1, c, s))
    assert torch.equal(lp, r.logprob) and torch.equal(ent, r.entropy) and torch.equal(tl, r.top_logprob) and torch.equal(ti, r.top_index)
    assert torch.equal(d, sc.grad)
    sc.grad = None
    loss, acc = class_nll(sc, lab)
    loss.backward()
    out, one = empty(3), torch.ones((), device=DEV)
    size = lib.mh_class_nll_workspace_bytes()
    ws = empty(size, dtype=torch.uint8)
    at = lambda t, i: ptr(t[i:])
    check(lib.mh_class_nll(ptr(sc), 0, 1, n, c, 0, 1, c, ptr(lab), -100, ptr(stat), at(out, 0), at(out, 1), at(out, 2), ptr(ws), size, s))
    check(lib.mh_class_nll_bwd(ptr(sc), 0, 1, n, c, 0, 1, c, ptr(lab), -100, ptr(stat), at(out, 2), ptr(one), ptr(d), 0, 1, c, s))
    assert float(out[0]) == float(loss.detach()) and float(out[1]) == float(acc) and torch.equal(d, sc.grad)


def test_group_norm_stays_in_bounds_for_graph_borders_that_do_not_ascend():
    """graph_ptr lies on the GPU and is not read on the host: borders that break its rule give rows of no defined value, and the
    kernels clamp what they read from it."""
    from magnet_amd.layer.norm import complex_group_norm
    n, f = 500, 8
    x = _features(n, f, seed=1).to(DEV)
    many = torch.randint(-1000, 2000, (3000,), generator=_gen(2)).to(torch.int32)
    for p in ([0, 400, 100, 500], [700, 3, -5, 2 ** 31 - 1], [5, 5, 5], many.tolist()):
        complex_group_norm(x, 2, graph_ptr=torch.tensor(p, device=DEV, dtype=torch.int32), relu=True)
        xr = x.clone().requires_grad_()
        complex_group_norm(xr, 2, graph_ptr=torch.tensor(p, device=DEV, dtype=torch.int32), checkpoint_bits=8).backward(x)
        torch.cuda.synchronize()
    want = complex_group_norm(x, 2)
    assert torch.equal(complex_group_norm(x, 2, graph_ptr=torch.tensor([0, n], device=DEV)), want)


def test_backward_of_a_kept_graph():
    """retain_graph: the norm, the scores and the GEMM-first convolution answer again; a convolution that let its orders go says so."""
    from magnet_amd import MagnetHipError
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.scores import class_nll
    from magnet_amd.layer.sparse_magnet import ChebConv
    from magnet_amd.utils.hermitian import ChebBasis
    x = _features(50, 8, seed=1).to(DEV).requires_grad_()
    y = complex_group_norm(x, 2, relu=True, checkpoint_bits=8)
    s = torch.randn(9, 4, device=DEV, requires_grad=True)
    loss, _ = class_nll(s, torch.zeros(9, dtype=torch.int64, device=DEV))
    for out, leaf in ((y.sum() + (y * y).sum(), x), (loss, s)):
        out.backward(retain_graph=True)
        first = leaf.grad.clone()
        leaf.grad = None
        out.backward()
        assert torch.equal(first, leaf.grad)
    with pytest.raises(RuntimeError, match='differentiated again'):
        g, = torch.autograd.grad(class_nll(s, torch.zeros(9, dtype=torch.int64, device=DEV))[0], s, create_graph=True)
        g.sum().backward()
    lap = _graph(60, 300)
    for cin, cout in ((8, 4), (4, 8)):
        conv = ChebConv(cin, cout, 2, ChebBasis(lap, 2), None).to(DEV)
        conv.checkpoint_bits = 8
        out = conv.forward_packed(_features(60, cin, seed=2).to(DEV)).sum()
        out.backward(retain_graph=True)
        first = conv.weight.grad.clone()
        conv.weight.grad = None
        if cout < cin:
            out.backward()
            assert torch.equal(first, conv.weight.grad)
        else:
            with pytest.raises(MagnetHipError, match='earlier backward'):
                out.backward()


def test_operators_share_a_gpu_between_streams_and_threads():
    """The same calls from two streams at once, each with workspaces of its own: the results of one after the other."""
    from magnet_amd.checkpoint import Checkpoint8
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.scores import class_nll
    n = 20000
    xs = [_features(n, 32, seed=k).to(DEV) for k in (1, 2)]
    ss = [torch.randn(1, 5, n, generator=_gen(k)).to(DEV) for k in (3, 4)]
    lab = torch.randint(0, 5, (1, n), generator=_gen(5)).to(DEV)

    def body(x, s):
        return [complex_group_norm(x, 4, relu=True), Checkpoint8.store(x).gram(x), *class_nll(s, lab)]

    want = [body(x, s) for x, s in zip(xs, ss)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(body(xs[i], ss[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_capture_beside_an_eager_pass_of_the_same_leaves():
    """The captured backward pass is refused where the leaves' accumulation lies on the default stream, and works once the eager
    pass is gone."""
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.scores import class_logprobs, class_nll
    n = 300
    x = _features(n, 8, seed=1).to(DEV).requires_grad_()
    w = torch.ones(8, device=DEV, requires_grad=True)
    v = torch.randn(n, 8, generator=_gen(2)).to(DEV).requires_grad_()
    lab = torch.randint(0, 8, (n,), generator=_gen(3)).to(DEV)
    leaves = (x, w, v)
    ones = {k: torch.ones(k, device=DEV) for k in ((n, 2, 8), (n,), ())}
    outs = (lambda: complex_group_norm(x * 2, 2, w, relu=True), lambda: class_nll(x[:, 0] + v, lab)[0],
            lambda: class_logprobs(x[:, 1] + v, lab, top=2).entropy)
    for out in outs:
        def backward():
            y = out()
            y.backward(ones[tuple(y.shape)])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            backward()                                             # the libraries' workspaces, the leaves' .grad
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        want = [t.grad.clone() for t in leaves if t.grad is not None]
        alive = out()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match='eager pass'):
            with torch.cuda.graph(graph):
                backward()
        torch.cuda.synchronize()
        alive.backward(ones[tuple(alive.shape)])                   # the eager pass itself is whole
        del alive, graph
        gc.collect()                                               # the error's frames
        for t in leaves:
            t.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            backward()
        for _ in range(3):
            for t in leaves:
                if t.grad is not None:
                    t.grad.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = [t.grad for t in leaves if t.grad is not None]
            assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
        del graph, got, want
        for t in leaves:
            t.grad = None
