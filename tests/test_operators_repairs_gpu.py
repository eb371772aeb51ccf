"""Norm, score and checkpoint operators at the places where an earlier form of them went wrong, against 64 bits on the CPU.

u = 2^-24 is the rounding of a float32 operation (half a step, relative).  Tolerances are worst-case counts of such roundings
along the formula."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------------------------
# gradients of single classes far below a row's largest
# ---------------------------------------------------------------------------------------------
# unit stride (pieces of 16 bytes), class-major with a lane or more for each row, four rows to a thread, strided, many classes
@pytest.mark.parametrize('rows,classes,layout', [(300, 5, 'row'), (300, 40, 'row'), (301, 7, 'class'), (70001, 5, 'class'), (65537, 8, 'class'),
                                                 (130, 12, 'strided'), (9, 1100, 'row'), (40, 100, 'class')])
def test_small_probabilities_have_their_own_accuracy(rows, classes, layout):
    """Every element of a gradient is as accurate as its own size asks, however small the class's probability is: scores are halves up
    to 31.5 on either side, so that x - m is exact."""
    from magnet_amd.layer.scores import class_logprobs, class_nll
    s = torch.randint(-63, 64, (rows, classes), generator=_gen(classes)).float() / 2
    lab = torch.randint(0, classes, (rows,), generator=_gen(rows))
    lp = torch.log_softmax(s.double(), 1)
    p, label = lp.exp(), lab.unsqueeze(1)
    if layout == 'class':
        given, labels = s.t().contiguous().unsqueeze(0).to(DEV), lab.unsqueeze(0).to(DEV)
    elif layout == 'strided':
        wide = torch.zeros(rows, 2 * classes + 1, device=DEV)
        wide[:, 1::2] = s.to(DEV)
        given, labels = wide[:, 1::2], lab.to(DEV)
    else:
        given, labels = s.to(DEV), lab.to(DEV)
    back = lambda t: t.detach().cpu()[0].t() if layout == 'class' else t.detach().cpu()
    # e^t: 2 u of the instruction and 2 u of its correction; a sum of `classes` terms, its additions and its terms' own errors (by
    # __expf, whose error of |t| 2 u against a share e^-|t| of the sum is below u of it); 2 u of its logarithm, which count as
    # 2 u log s in e^-log s, 4 u of that; two products and 1 / rows
    rel = (2 * classes + 20 + 2 * math.log(classes)) * U
    far = ~torch.zeros(rows, classes, dtype=torch.bool).scatter(1, label, True)
    t = given.detach().requires_grad_()
    class_nll(t, labels)[0].backward()
    got, want = back(t.grad).double(), p / rows
    assert float(((got - want).abs() / want)[far].max()) <= rel
    t = given.detach().requires_grad_()
    class_logprobs(t, labels).logprob.sum().backward()
    got = back(t.grad).double()
    assert float(((got + p).abs() / p)[far].max()) <= rel


# ---------------------------------------------------------------------------------------------
# convolutions with 8-bit checkpoints
# ---------------------------------------------------------------------------------------------
def _conv(cin, cout, n, k=2, bits=8):
    from magnet_amd.laplacian import build_magnetic_laplacian, powerlaw_edges
    from magnet_amd.layer.sparse_magnet import ChebConv
    from magnet_amd.utils.hermitian import ChebBasis
    src, dst = powerlaw_edges(n, 3 * n, 3, device=DEV)
    torch.manual_seed(0)
    conv = ChebConv(cin, cout, k, ChebBasis(build_magnetic_laplacian(src, dst, n, q=0.15), k), None).to(DEV)
    conv.checkpoint_bits = bits
    return conv


@pytest.mark.parametrize('cin,cout', [(64, 16), (16, 64)])
def test_a_backward_pass_lets_its_checkpoint_go(cin, cout):
    """What a convolution kept is gone behind its backward pass, also while the loss that led there lives on."""
    n, left = 20000, {}
    for bits in (32, 8):
        conv = _conv(cin, cout, n, bits=bits)
        x = torch.randn(n, 2, cin, generator=_gen(1)).to(DEV)
        conv.forward_packed(x).sum().backward()                    # plans, library handles, the gradients' memory
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = conv.forward_packed(x, relu=True).sum()
        kept = torch.cuda.memory_allocated() - before
        loss.backward()
        left[bits] = torch.cuda.memory_allocated() - before
        assert bits == 32 or kept >= 2 * n * cin                   # the codes at least; in 32 bits it may be x itself
        del loss
    # the allocator rounds to 512 bytes, a handful of tensors
    assert left[8] <= left[32] + 4096, left


# ---------------------------------------------------------------------------------------------
# what a loss keeps
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize('rows,classes', [(2500, 5), (300000, 5), (300000, 40)])
def test_a_loss_keeps_what_its_backward_pass_reads(rows, classes):
    """Nothing for each row where the backward pass makes it again; through raw pointers with no memory for it, the same gradient."""
    from magnet_amd._lib import lib, ptr, stream_ptr, check
    from magnet_amd.layer.scores import class_nll
    s = torch.randn(1, classes, rows, generator=_gen(1)).to(DEV).requires_grad_()
    lab = torch.randint(0, classes, (1, rows), generator=_gen(2)).to(DEV)
    class_nll(s, lab)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss, _ = class_nll(s, lab)
    kept = torch.cuda.memory_allocated() - before
    size = lib.mh_class_nll_stat_bytes(1, rows, classes, rows, 1)
    assert (size == 0) == (rows > 10000 and classes == 5) and kept <= size + 4096, (kept, size)
    loss.backward()
    if size == 0:
        out, one, d = torch.empty(3, device=DEV), torch.ones((), device=DEV), torch.empty_like(s)
        bytes_ = lib.mh_class_nll_workspace_bytes()
        ws, st = torch.empty(bytes_, dtype=torch.uint8, device=DEV), stream_ptr(torch.device(DEV, 0))
        args = (ptr(s), 0, 1, rows, classes, 0, rows, 1, ptr(lab), -100, None)
        check(lib.mh_class_nll(*args, ptr(out), ptr(out[1:]), ptr(out[2:]), ptr(ws), bytes_, st))
        check(lib.mh_class_nll_bwd(*args, ptr(out[2:]), ptr(one), ptr(d), 0, rows, 1, st))
        assert float(out[0]) == float(loss.detach()) and torch.equal(d, s.grad)


@pytest.mark.parametrize('rows', [2500, 65536, 70001])
def test_a_gradient_of_zero_reaches_no_row(rows):
    """A loss that counts for nothing has gradients of 0, in every kernel: also for a row without a distribution, and NaN for a
    label out of range."""
    from magnet_amd.layer.scores import class_nll
    s = torch.randn(1, 5, rows, generator=_gen(1))
    s[0, :, 7], s[0, 2, 9], s[0, 1, 11] = -float('inf'), float('nan'), float('inf')
    lab = torch.randint(0, 5, (1, rows), generator=_gen(2))
    lab[0, 20] = 5
    s = s.to(DEV).requires_grad_()
    class_nll(s, lab.to(DEV))[0].backward(torch.zeros((), device=DEV))
    wrong = torch.zeros(rows, dtype=torch.bool)
    wrong[20] = True
    d = s.grad.cpu()[0]
    assert bool(torch.isnan(d[:, wrong]).all()) and not bool(d[:, ~wrong].any()) and not bool(torch.isnan(d[:, ~wrong]).any())


# ---------------------------------------------------------------------------------------------
# group norm
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_a_gradient_that_is_not_finite_shows_behind_a_closed_gate(bits, value):
    """The joined gate multiplies, as complex_relu_layer does behind a convolution: the same elements are NaN as in a norm and a
    layer of their own."""
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.sparse_magnet import _ComplexReluFn
    x = torch.randn(50, 2, 8, generator=_gen(1)).to(DEV)
    w = torch.ones(8, device=DEV)
    ptr = torch.tensor([0, 20, 50], dtype=torch.int32, device=DEV)
    closed = torch.nonzero(complex_group_norm(x, 2, graph_ptr=ptr)[:20, 0] < 0)[0]
    g = torch.randn(50, 2, 8, generator=_gen(2)).to(DEV)
    g[closed[0], 1, closed[1]] = value
    grads = []
    for joined in (True, False):
        xr, wr, br = (t.clone().requires_grad_() for t in (x, w, torch.zeros_like(w)))
        y = complex_group_norm(xr, 2, wr, br, graph_ptr=ptr, relu=joined, checkpoint_bits=bits)
        (y if joined else _ComplexReluFn.apply(y)).backward(g)
        grads.append((xr.grad, wr.grad, br.grad))
    for a, b in zip(*grads):
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and bool(torch.isnan(b).any())
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize('n,f,groups,relu,bits', [(300007, 30, 5, False, 32), (200001, 30, 5, True, 8)])
def test_group_norm_of_a_large_graph_with_odd_channels(n, f, groups, relu, bits):
    """Two channels to a thread, sums over a million values, against the definition evaluated on the CPU."""
    import test_operators_gpu as T
    from magnet_amd.layer.norm import complex_group_norm
    x, g = T._features(n, f, seed=n), torch.randn(n, 2, f, generator=_gen(5)) / n
    w, b = 0.5 + torch.rand(f, generator=_gen(f)), torch.rand(f, generator=_gen(f + 1)) - 0.3
    x = T._off_the_gate(x, groups, w.double(), b.double(), [n], 1e-5) if relu else x
    held = torch.from_numpy(T._restored(x)) if bits == 8 else None
    out, dx, dw, db, tol_out, tol_dx, mag_w, mag_b = T._norm_reference(x, groups, w.double(), b.double(), [n], 1e-5, relu, g, held)
    xd, wd, bd = (t.to(DEV).requires_grad_() for t in (x, w, b))
    y = complex_group_norm(xd, groups, wd, bd, relu=relu, checkpoint_bits=bits)
    y.backward(g.to(DEV))
    # the same counts of roundings as for the small graphs: sums are held in 64 bits
    T._close(y.detach(), out, 8 * U * tol_out + 1e-300, 'result')
    T._close(xd.grad, dx, 20 * U * tol_dx + 1e-300, 'dx')
    T._close(wd.grad, dw, 8 * U * mag_w + 1e-300, 'dweight')
    T._close(bd.grad, db, 4 * U * mag_b + 1e-300, 'dbias')
    # over all values together: each is within a few roundings, so their norm is
    assert float((y.detach().double().cpu() - out).norm() / out.norm()) < 2 * U


# ---------------------------------------------------------------------------------------------
# the C ABI without torch
# ---------------------------------------------------------------------------------------------
def test_operators_from_a_plain_cpp_caller():
    """tests/abi/abi_operators.cpp: the checkpoint, norm and score entry points called from plain C++, results against their
    formulas in double precision on the host, the memory behind every output untouched."""
    import os
    import subprocess
    from conftest import ROOT
    exe = os.path.join(ROOT, 'tests', 'abi', 'abi_operators')
    assert os.path.isfile(exe), 'tests/abi/abi_operators is not built (make -C magnet_amd/csrc)'
    res = subprocess.run([exe], capture_output=True, text=True, timeout=110)
    assert res.returncode == 0 and res.stdout.strip().endswith('operators ok'), (res.stdout[-300:], res.stderr[-3000:])


# ---------------------------------------------------------------------------------------------
# offsets that pass 32 bits
# ---------------------------------------------------------------------------------------------
def _wide_gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def test_checkpoints_of_more_than_2_to_32_values():
    """4.6G values: both ends byte for byte as on their own; the weight gradient as the sum of its halves (all terms positive, so
    that a bound of 12288 float32 additions is one of the result)."""
    from magnet_amd.checkpoint import Checkpoint8
    n, m, k, ends = 6_000_000, 384, 8, 1001
    x = torch.rand(n, 2, m, device=DEV, generator=_wide_gen(1))
    g = torch.rand(n, 2, k, device=DEV, generator=_wide_gen(2))
    ck = Checkpoint8.store(x)
    assert ck.codes.numel() > 2 ** 32
    for part, rows in ((slice(0, ends), slice(0, 2 * ends)), (slice(n - ends, n), slice(2 * (n - ends), 2 * n))):
        own = Checkpoint8.store(x[part])
        assert torch.equal(own.codes, ck.codes[rows]) and torch.equal(own.scales[:, :2 * ends], ck.scales[:, rows])
    back = ck.restore()
    for part in (slice(0, ends), slice(n - ends, n)):
        assert torch.equal(back[part], Checkpoint8.store(x[part]).restore())
    del back
    halves = sum(Checkpoint8.store(x[part]).gram(g[part]).double() for part in (slice(0, n // 2), slice(n // 2, n)))
    got = ck.gram(g).double()
    assert float(((got - halves).abs() / halves).max()) <= 2 * (12288 + 8) * U


@pytest.mark.parametrize('bits', [32, 8])
def test_group_norm_of_more_than_2_to_31_values(bits):
    """The last graph of 2.3G values, forward and backward, as on its own."""
    from magnet_amd.layer.norm import complex_group_norm
    n, f, last = 9_000_000, 128, 10007
    x = torch.randn(n, 2, f, device=DEV, generator=_wide_gen(1)).requires_grad_()
    g = torch.randn(n, 2, f, device=DEV, generator=_wide_gen(2))
    ptr = torch.tensor([0, n - last, n], dtype=torch.int32, device=DEV)
    y = complex_group_norm(x, 8, graph_ptr=ptr, relu=True, checkpoint_bits=bits)
    y.backward(g)
    own = x[n - last:].detach().requires_grad_()
    z = complex_group_norm(own, 8, relu=True, checkpoint_bits=bits)
    z.backward(g[n - last:])
    y, z = y.detach(), z.detach()
    # the same formula on the same values, its 64-bit sums in another order: a rounding of mean and deviation either way; a gate
    # that opens with it is 0 on one side
    same = (y[n - last:, :1] == 0) == (z[:, :1] == 0)
    assert float((~same).sum()) <= 8
    assert float(((y[n - last:] - z).abs() * same).max()) <= 16 * U * float(z.abs().max())
    assert float(((x.grad[n - last:] - own.grad).abs() * same).max()) <= 64 * U * float(own.grad.abs().max())
    assert bool(torch.isfinite(y[::4999]).all()) and bool(torch.isfinite(x.grad[::4999]).all())


@pytest.mark.parametrize('rows,classes,layout,dtype', [(60_000_000, 40, 'class', torch.float32), (7_000_000, 349, 'row', torch.bfloat16),
                                                       (300_000_000, 8, 'class', torch.bfloat16)])
def test_scores_of_more_than_2_to_31_values(rows, classes, layout, dtype):
    """The last rows as on their own; the loss as the mean of its halves."""
    from magnet_amd.layer.scores import class_logprobs, class_nll
    end, by_class = 1003, layout == 'class'
    s = torch.empty((1, classes, rows) if by_class else (rows, classes), device=DEV, dtype=dtype).normal_(generator=_wide_gen(1)).requires_grad_()
    lab = torch.randint(0, classes, (1, rows) if by_class else (rows,), device=DEV, generator=_wide_gen(2))
    assert s.numel() > 2 ** 31
    tail = lambda t: t[..., rows - end:] if by_class else t[rows - end:]
    own = tail(s).detach().contiguous().requires_grad_()
    loss, acc = class_nll(s, lab)
    loss.backward()
    part, _ = class_nll(own, tail(lab).contiguous())
    (part * (end / rows)).backward()
    depth = (classes + 32) * U + torch.finfo(dtype).eps              # two values a rounding apart may be two steps of the type apart
    assert float((tail(s.grad).double() - own.grad.double()).abs().max()) <= depth / rows
    loss = loss.detach()
    halves = [class_nll(t.detach(), u) for t, u in ((s[..., :rows // 2], lab[..., :rows // 2]), (s[..., rows // 2:], lab[..., rows // 2:]))] \
        if by_class else [class_nll(t.detach(), u) for t, u in zip(s.split(rows // 2), lab.split(rows // 2))]
    assert abs(float(loss) - float(halves[0][0] + halves[1][0]) / 2) <= 8 * U * float(loss)
    assert abs(float(acc) - float(halves[0][1] + halves[1][1]) / 2) <= 8 * U
    s.grad = None
    r, q = class_logprobs(s.detach(), lab, top=2), class_logprobs(own.detach(), tail(lab).contiguous(), top=2)
    for a, b in ((tail(r.logprob), q.logprob), (tail(r.entropy), q.entropy)):
        assert float((a - b).abs().max()) <= depth * 16
    assert torch.equal(r.top_index[..., rows - end:] if by_class else r.top_index[rows - end:], q.top_index)
