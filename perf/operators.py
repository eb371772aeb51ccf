"""The operators of a memory-lean training step, and the cases they are measured at.

nll    mean negative log-likelihood and accuracy of class scores, with the gradient of the scores (node and link heads)
report log probability of a given class, entropy and top alternatives of every row; `grad` adds the gradient of the scores
norm   complex group norm of row-planar features [N, 2, F] over the graphs of a batch, optional complex ReLU; `train` adds the
       gradients; `bits` 8 keeps the input for the backward pass in 8 bits
keep   an activation checkpoint in 8 bits: stored and restored
gram   the weight gradient A^T G of a convolution whose propagated features A are held as such a checkpoint

`own` false: plain torch operations.  `own` true: the calls of magnet_amd.
"""
import math

import torch

own = False

DEV = 'cuda'
IGNORE = -100
BLOCK = 32                     # columns that share one power-of-two scale in a checkpoint
EPS = 1e-5
SLAB = 16384                   # rows of one product of the plain weight gradient
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # a driver's own dataset (2500 nodes, 5 classes): one training step's loss, bound by launches
        dict(name='nll-node-small', op='nll', rows=2500, classes=5, layout='class', type='f32'),
        # the benchmark's epoch: 2M nodes, class-major scores as the head writes them
        dict(name='nll-node-graph', op='nll', rows=2_000_000, classes=5, layout='class', type='f32'),
        # link prediction: pairs scored row by row, an evaluation report with two alternatives
        dict(name='report-links', op='report', rows=300_001, classes=3, layout='row', type='f32', top=2, grad=False),
        # many classes in half precision, training on the log probability with an entropy term
        dict(name='report-wide-train', op='report', rows=60_001, classes=349, layout='row', type='bf16', top=5, grad=True),
        # a driver's own dataset: 16 filters in 4 groups, a training step's pass
        dict(name='norm-small', op='norm', nodes=2500, graphs=1, feats=16, groups=4, relu=True, train=True, bits=32),
        # a large graph, 128 filters: the bandwidth case
        dict(name='norm-graph', op='norm', nodes=1_000_000, graphs=1, feats=128, groups=8, relu=True, train=True, bits=32),
        # a batch of ragged graphs, empty ones among them, the saved input in 8 bits
        dict(name='norm-batch-8bit', op='norm', nodes=200_003, graphs=512, feats=64, groups=8, relu=True, train=True, bits=8),
        # an evaluation forward at a width that no vector divides
        dict(name='norm-eval-odd', op='norm', nodes=300_007, graphs=1, feats=30, groups=5, relu=False, train=False, bits=32),
        # the K + 1 = 3 orders of a 128-filter convolution kept and read back
        dict(name='keep-orders', op='keep', nodes=500_000, cols=384),
        # weight gradient of a driver-sized convolution (16 filters, K = 2)
        dict(name='gram-small', op='gram', nodes=2500, cols=48, out=16),
        # an odd width: K + 1 = 4 orders of 30 filters
        dict(name='gram-odd', op='gram', nodes=150_001, cols=120, out=30),
        # weight gradient of a 128-filter convolution, K = 2, on a large graph
        dict(name='gram-graph', op='gram', nodes=1_000_000, cols=384, out=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('nll', 'report', 'norm', 'norm', 'keep', 'gram', 'gram'))
    if op == 'nll':
        classes = _log_int(rng, 2, 70)
        return dict(op=op, rows=_log_int(rng, 1, 10_000_000 // classes), classes=classes, layout=rng.choice(('class', 'row')),
                    type=rng.choice(('f32', 'f32', 'bf16', 'f16')))
    if op == 'report':
        classes = _log_int(rng, 2, 2000)
        return dict(op=op, rows=_log_int(rng, 1, 8_000_000 // classes), classes=classes, layout=rng.choice(('class', 'row', 'row')),
                    type=rng.choice(('f32', 'bf16', 'f16')), top=rng.randint(0, min(8, classes)), grad=rng.random() < 0.5)
    if op == 'norm':
        groups = rng.choice((1, 2, 3, 5, 8, 16))
        feats = groups * _log_int(rng, 1, max(1, 256 // groups))
        nodes = _log_int(rng, 1, 100_000_000 // feats if feats > 100 else 1_000_000)
        graphs = 1 if rng.random() < 0.5 else _log_int(rng, 1, min(2000, nodes))
        train = rng.random() < 0.7
        return dict(op=op, nodes=nodes, graphs=graphs, feats=feats, groups=groups, relu=rng.random() < 0.6, train=train,
                    bits=rng.choice((32, 32, 8)) if train else 32)
    if op == 'keep':
        cols = _log_int(rng, 1, 1024)
        return dict(op=op, nodes=_log_int(rng, 1, min(1_500_000, 180_000_000 // cols)), cols=cols)
    cols, out = _log_int(rng, 1, 1024), _log_int(rng, 1, 256)
    most = min(1_500_000, 45_000_000_000 // (cols * out), 180_000_000 // (cols + out))
    return dict(op=op, nodes=_log_int(rng, 1, most), cols=cols, out=out)


def work(case):
    op = case['op']
    if op in ('nll', 'report'):
        n, c = case['rows'], case['classes']
        e = 4 if case['type'] == 'f32' else 2
        if op == 'nll':
            return dict(bytes=2 * e * n * c + 8 * n, flops=10 * n * c)
        grads = (e * n * c + 8 * n) if case['grad'] else 0
        return dict(bytes=e * n * c + 8 * n + 8 * n + 12 * n * case['top'] + grads, flops=(16 if case['grad'] else 8) * n * c)
    if op == 'norm':
        v = 2 * case['nodes'] * case['feats']
        return dict(bytes=(16 if case['train'] else 8) * v + 12 * case['feats'], flops=(24 if case['train'] else 8) * v)
    rows = 2 * case['nodes']
    if op == 'keep':
        return dict(bytes=8 * rows * case['cols'], flops=4 * rows * case['cols'])
    m, n = case['cols'], case['out']
    return dict(bytes=rows * m + rows * -(-m // BLOCK) + 4 * rows * n + 4 * m * n, flops=2 * rows * m * n)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _graph_sizes(nodes, graphs, seed):
    """Sizes of the graphs of a batch: ragged over two orders of magnitude, one in ten empty; they sum to `nodes`."""
    if graphs == 1:
        return torch.tensor([nodes])
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(torch.rand(graphs, generator=g) * 4.6)
    w[torch.rand(graphs, generator=g) < 0.1] = 0.0
    w[0] = 1.0
    edges = torch.floor(torch.cumsum(w.double(), 0) / w.double().sum() * nodes + 0.5).long()
    edges[-1] = nodes
    return torch.diff(torch.cat([torch.zeros(1, dtype=torch.long), edges]))


def _features(nodes, parts, cols, gen):
    """Aggregated features: rows of different magnitude (hub nodes are large), channels with offsets of their own."""
    x = torch.randn(nodes, parts, cols, device=DEV, generator=gen)
    x.mul_(torch.exp(0.5 * torch.randn(nodes, 1, 1, device=DEV, generator=gen)))
    return x.add_(0.7 * torch.randn(1, parts, cols, device=DEV, generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, st = case['op'], dict(case)
    if op in ('nll', 'report'):
        n, c = case['rows'], case['classes']
        shape = (1, c, n) if case['layout'] == 'class' else (n, c)
        st['scores'] = (3.0 * torch.randn(shape, device=DEV, generator=gen)).to(TYPES[case['type']])
        rows = (1, n) if case['layout'] == 'class' else (n,)
        lab = torch.randint(0, c, rows, device=DEV, generator=gen)
        # a training split: the other nodes carry the ignored label
        st['labels'] = torch.where(torch.rand(rows, device=DEV, generator=gen) < 0.4, torch.full_like(lab, IGNORE), lab)
        st['labels'].view(-1)[0] = c - 1
        if op == 'report' and case['grad']:
            st['g_logprob'] = torch.randn(rows, device=DEV, generator=gen) / n
            st['g_entropy'] = torch.randn(rows, device=DEV, generator=gen) * (0.1 / n)
        return st
    if op == 'norm':
        n, f = case['nodes'], case['feats']
        sizes = _graph_sizes(n, case['graphs'], seed)
        ptr = torch.zeros(len(sizes) + 1, dtype=torch.int32)
        ptr[1:] = torch.cumsum(sizes, 0)
        st['ptr'] = ptr.to(DEV) if case['graphs'] > 1 else None
        st['x'] = _features(n, 2, f, gen)
        st['weight'] = 0.5 + torch.rand(f, device=DEV, generator=gen)
        st['bias'] = 0.3 * torch.randn(f, device=DEV, generator=gen)
        if case['relu']:
            # a value on the border of the gate is decided by the last bit of any arithmetic: such values are moved off it
            y = _normed(st['x'], case['groups'], st['ptr'])[0][:, 0].double() * st['weight'] + st['bias']
            st['x'][:, 0] += 0.05 * (y.abs() < 1e-4)
            del y
        if case['train']:
            st['g'] = torch.randn(n, 2, f, device=DEV, generator=gen) * (1.0 / n)
        return st
    n, m = case['nodes'], case['cols']
    x = _features(n, 2, m, gen)
    if op == 'keep':
        st['x'] = x
        return st
    # what the forward pass left: codes and scales; and the gradient of the convolution's output, half of it gated away
    st['codes'], st['scales'] = _held(x)
    del x
    k = case['out']
    g = torch.randn(n, 2, k, device=DEV, generator=gen) * (1.0 / n)
    st['g'] = g * (torch.rand(n, 1, k, device=DEV, generator=gen) < 0.5)
    return st


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _blocks(x):
    """[N, 2, m] -> [2N, blocks, 32], the last block filled up with zeros."""
    n, parts, m = x.shape
    return torch.nn.functional.pad(x.reshape(n * parts, m), (0, -m % BLOCK)).view(n * parts, -1, BLOCK)


def _quantised(x):
    """Integers in -127 .. 127 and the exponent of the scale of each block of 32 columns."""
    b = _blocks(x)
    top = b.abs().amax(-1)
    mant, expo = torch.frexp(top)
    e = torch.where(torch.round(mant * 128.0) > 127.0, expo - 6, expo - 7).clamp(-110, 121)
    q = torch.round(torch.ldexp(b, -e.unsqueeze(-1))).clamp(-127, 127)
    return q, e


def _held(x):
    """The bytes of a checkpoint: codes [2N, columns up to a multiple of 32], the integers + 128, and scale exponents + 128,
    [blocks, 2N up to a multiple of 8], the rows behind the last filled with 0 and every code there unused."""
    q, e = _quantised(x)
    rows = q.size(0)
    codes = (q + 128).to(torch.uint8).view(rows, -1)
    scales = torch.zeros(e.size(1), -(-rows // 8) * 8, dtype=torch.uint8, device=x.device)
    scales[:, :rows] = (e + 128).t().to(torch.uint8)
    return codes, scales


def _values(codes, scales, m):
    """[2N, m] float32 values that the bytes stand for."""
    rows = codes.size(0)
    q = codes.to(torch.float32).view(rows, -1, BLOCK) - 128.0
    e = scales[:, :rows].t().to(torch.int32) - 128
    return torch.ldexp(q, e.unsqueeze(-1)).view(rows, -1)[:, :m]


def _graph_of_row(ptr, n):
    return torch.searchsorted(ptr[1:].contiguous(), torch.arange(n, device=ptr.device, dtype=ptr.dtype), right=True)


def _graph_sums(v, ptr):
    """Sums of v [N, ...] (64 bits) over the rows of each graph."""
    if ptr is None:
        return v.sum(0, keepdim=True)
    ahead = torch.nn.functional.pad(torch.cumsum(v.flatten(1).t().contiguous(), 1), (1, 0))[:, ptr.long()]
    return torch.diff(ahead).t().reshape((-1,) + tuple(v.shape[1:]))


def _rows(v, ptr, n):
    """Per-graph values v [B, ...] at each row."""
    return v if ptr is None else v[_graph_of_row(ptr, n)]


def _normed(x, groups, ptr):
    """(normalised features, mean, 1 / deviation [rows, 1, G, 1], M [rows, 1]): statistics in 64 bits, the rest in 32."""
    n, _, f = x.shape
    d = f // groups
    v = x.view(n, 2, groups, d)
    sizes = torch.diff(ptr).double().view(-1, 1) if ptr is not None else torch.full((1, 1), float(n), dtype=torch.float64, device=x.device)
    count = sizes.clamp(min=1.0) * d
    mean = _graph_sums(v.sum(3, dtype=torch.float64), ptr) / count.unsqueeze(1)
    centred = v - _rows(mean.float(), ptr, n).unsqueeze(-1)
    var = _graph_sums((centred * centred).sum((1, 3), dtype=torch.float64), ptr) / count
    rstd = _rows((1.0 / torch.sqrt(var + EPS)).float(), ptr, n).view(-1, 1, groups, 1)
    return (centred * rstd).view(n, 2, f), mean, rstd, _rows(count, ptr, n)


def _plain_norm(st):
    x, w, b, ptr, groups = st['x'], st['weight'], st['bias'], st['ptr'], st['groups']
    n, _, f = x.shape
    xh, mean, rstd, count = _normed(x, groups, ptr)
    y = xh * w + b
    keep = (y[:, :1] >= 0).float() if st['relu'] else None
    out = y * keep if st['relu'] else y
    if not st['train']:
        return out
    if st['bits'] == 8:
        q, e = _quantised(x)
        held = torch.ldexp(q, e.unsqueeze(-1)).view(n, 2, -1)[:, :, :f]
        xh = ((held.view(n, 2, groups, -1) - _rows(mean.float(), ptr, n).unsqueeze(-1)) * rstd).view(n, 2, f)
    dy = st['g'] * keep if st['relu'] else st['g']
    dw = (dy * xh).sum((0, 1), dtype=torch.float64).float()
    db = dy.sum((0, 1), dtype=torch.float64).float()
    dxh = (dy * w).view(n, 2, groups, -1)
    flat = _rows(_graph_sums(dxh.sum(3, dtype=torch.float64), ptr), ptr, n) / count.unsqueeze(1)
    along = _rows(_graph_sums((dxh * xh.view_as(dxh)).sum((1, 3), dtype=torch.float64), ptr), ptr, n) / count
    dx = rstd * (dxh - flat.float().unsqueeze(-1) - xh.view_as(dxh) * along.float().view(-1, 1, groups, 1))
    return out, dx.view(n, 2, f), dw, db


def _class_first(st):
    """Scores [C, rows] in 32 bits and labels [rows]."""
    s = st['scores'].float()
    return (s[0] if st['layout'] == 'class' else s.t()), st['labels'].view(-1)


def _as_given(d, st):
    return (d.unsqueeze(0) if st['layout'] == 'class' else d.t().contiguous()).to(TYPES[st['type']])


def _log_softmax(s):
    z = s - s.amax(0, keepdim=True)
    return z - torch.log(torch.exp(z).sum(0, keepdim=True))


def _plain_nll(st):
    s, lab = _class_first(st)
    lp = _log_softmax(s)
    use = lab != IGNORE
    one = torch.arange(s.size(0), device=s.device).unsqueeze(1) == lab
    count = use.sum()
    loss = -(torch.where(one, lp, 0.0).sum(0).sum(dtype=torch.float64) / count).float()
    hits = ((s.argmax(0) == lab).sum().double() / count).float()
    ds = torch.where(use, (torch.exp(lp) - one.float()) / count, 0.0)
    return loss, hits, _as_given(ds, st)


def _plain_report(st):
    s, lab = _class_first(st)
    lp = _log_softmax(s)
    p = torch.exp(lp)
    one = torch.arange(s.size(0), device=s.device).unsqueeze(1) == lab
    of_label = torch.where(one, lp, 0.0).sum(0)
    entropy = -(p * lp).sum(0)
    k = st['top']
    order = torch.sort(s, dim=0, descending=True, stable=True)[1][:k]
    top = torch.gather(lp, 0, order)
    by_class = st['layout'] == 'class'
    out = [of_label.view(st['labels'].shape), entropy.view(st['labels'].shape)]
    out += [top.unsqueeze(0) if by_class else top.t().contiguous(), order.unsqueeze(0) if by_class else order.t().contiguous()]
    if st['grad']:
        gl = torch.where(lab != IGNORE, st['g_logprob'].view(-1), 0.0)
        out.append(_as_given(gl * (one.float() - p) - st['g_entropy'].view(-1) * p * (lp + entropy), st))
    return out


def _plain(st):
    op = st['op']
    if op == 'nll':
        return _plain_nll(st)
    if op == 'report':
        return _plain_report(st)
    if op == 'norm':
        return _plain_norm(st)
    if op == 'keep':
        codes, scales = _held(st['x'])
        return _values(codes, scales, st['cols']).view(st['x'].shape)
    # slabs of rows as one batched product, their results summed: a single sum over millions of rows in 32 bits loses digits
    m, k = st['cols'], st['out']
    a, g = _values(st['codes'], st['scales'], m), st['g'].view(-1, k)
    more = (0, 0, 0, -a.size(0) % SLAB) if a.size(0) > SLAB else (0, 0)
    a, g = torch.nn.functional.pad(a, more), torch.nn.functional.pad(g, more)
    slab = min(SLAB, a.size(0))
    return torch.bmm(a.view(-1, slab, m).transpose(1, 2), g.view(-1, slab, k)).sum(0)


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------
def _framework(st):
    op = st['op']
    if op in ('nll', 'report'):
        from magnet_amd.layer.scores import class_logprobs, class_nll
        grad = op == 'nll' or st['grad']
        s = st['scores'].detach().requires_grad_(grad)
        if op == 'nll':
            loss, accuracy = class_nll(s, st['labels'])
            loss.backward()
            return loss.detach(), accuracy, s.grad
        r = class_logprobs(s, st['labels'], top=st['top'])
        out = [r.logprob.detach(), r.entropy.detach(), r.top_logprob.detach(), r.top_index]
        if grad:
            torch.autograd.backward([r.logprob, r.entropy], [st['g_logprob'], st['g_entropy']])
            out.append(s.grad)
        return out
    if op == 'norm':
        from magnet_amd.layer.norm import complex_group_norm
        train = st['train']
        x, w, b = (st[k].detach().requires_grad_(train) for k in ('x', 'weight', 'bias'))
        y = complex_group_norm(x, st['groups'], w, b, graph_ptr=st['ptr'], eps=EPS, relu=st['relu'], checkpoint_bits=st['bits'])
        if not train:
            return y
        y.backward(st['g'])
        return y.detach(), x.grad, w.grad, b.grad
    from magnet_amd.checkpoint import Checkpoint8
    if op == 'keep':
        return Checkpoint8.store(st['x']).restore()
    return Checkpoint8(st['codes'], st['scales'], (st['nodes'], 2, st['cols'])).gram(st['g'])


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_scores(case, st):
    s = st['scores'].double().requires_grad_()
    lab = st['labels']
    rows = (s.permute(0, 2, 1) if case['layout'] == 'class' else s).reshape(-1, case['classes'])
    flat = lab.reshape(-1)
    lse = torch.logsumexp(rows, 1)
    use = flat >= 0
    of_label = torch.where(use, rows.gather(1, flat.clamp(min=0).unsqueeze(1)).squeeze(1) - lse, 0.0)
    if case['op'] == 'nll':
        loss = -of_label.sum() / use.sum()
        grad, = torch.autograd.grad(loss, s)
        best = rows.detach().max(1, keepdim=True)[0]
        place = torch.arange(case['classes'], device=DEV).expand_as(rows)
        first = torch.where(rows.detach() == best, place, case['classes']).amin(1)
        return loss.detach(), ((first == flat) & use).sum().double() / use.sum(), grad
    entropy = torch.special.entr(torch.exp(rows - lse.unsqueeze(1))).sum(1)
    k = case['top']
    best = torch.topk(rows.detach(), k, dim=1)[0] - lse.detach().unsqueeze(1)
    best = best.t().unsqueeze(0) if case['layout'] == 'class' else best
    out = [of_label.detach().view(lab.shape), entropy.detach().view(lab.shape), best, None]
    if case['grad']:
        total = (of_label * st['g_logprob'].double().view(-1)).sum() + (entropy * st['g_entropy'].double().view(-1)).sum()
        out.append(torch.autograd.grad(total, s)[0])
    return out


def _exact_held(x):
    """x [N, 2, m] -> the nearest value of code * 2^s, by the definition of the format, in 64 bits."""
    n, _, m = x.shape
    out = torch.empty(n, 2, m, dtype=torch.float64, device=x.device)
    for c in range(0, m, BLOCK):
        v = x[:, :, c:c + BLOCK].double()
        top = v.abs().amax(2, keepdim=True)
        p = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) + 1
        p = torch.where(top >= torch.exp2(p), p + 1, torch.where(top < torch.exp2(p - 1), p - 1, p))
        p = torch.where(torch.round(top * torch.exp2(7 - p)) > 127, p + 1, p)
        step = torch.exp2((p - 7).clamp(-110, 121))
        out[:, :, c:c + BLOCK] = (v / step).round().clamp(-127, 127) * step
    return out


def _exact_norm(case, st):
    groups, f = case['groups'], case['feats']
    sizes = [case['nodes']] if st['ptr'] is None else torch.diff(st['ptr']).tolist()
    w, b = st['weight'].double(), st['bias'].double()
    held = _exact_held(st['x']) if case['train'] and case['bits'] == 8 else None
    outs, dxs, dw, db, at = [], [], torch.zeros_like(w), torch.zeros_like(b), 0
    for n in sizes:
        x = st['x'][at:at + n].double()
        if n:
            z = torch.complex(x[:, 0], x[:, 1]).view(n, groups, -1)
            mean = z.mean((0, 2), keepdim=True)
            sd = torch.sqrt((z - mean).abs().square().mean((0, 2), keepdim=True) + EPS)
            y = ((z - mean) / sd).view(n, f) * w + torch.complex(b, b)
            gate = (y.real >= 0).double() if case['relu'] else torch.ones_like(y.real)
            y = y * gate
            outs.append(torch.stack((y.real, y.imag), 1))
            if case['train']:
                if held is not None:
                    z = torch.complex(held[at:at + n, 0], held[at:at + n, 1]).view(n, groups, -1)
                g = st['g'][at:at + n].double()
                dy = torch.complex(g[:, 0], g[:, 1]) * gate
                zn = ((z - mean) / sd).view(n, f)
                inner = (dy * zn.conj()).real
                dw += inner.sum(0)
                db += (dy.real + dy.imag).sum(0)
                dz = (dy * w).view(n, groups, -1)
                pull = (inner * w).view(n, groups, -1).mean((0, 2), keepdim=True)
                dz = ((dz - dz.mean((0, 2), keepdim=True) - zn.view(n, groups, -1) * pull) / sd).view(n, f)
                dxs.append(torch.stack((dz.real, dz.imag), 1))
        at += n
    out = torch.cat(outs)
    return (out, torch.cat(dxs), dw, db) if case['train'] else out


def exact(case, seed):
    st = prepare(case, seed)
    op = case['op']
    if op in ('nll', 'report'):
        return _exact_scores(case, st)
    if op == 'norm':
        return _exact_norm(case, st)
    if op == 'keep':
        return _exact_held(st['x'])
    rows, m, k = 2 * case['nodes'], case['cols'], case['out']
    g = st['g'].view(rows, k)
    total = torch.zeros(m, k, dtype=torch.float64, device=DEV)
    for r in range(0, rows, 1 << 19):
        q = st['codes'][r:r + (1 << 19), :m].double() - 128
        two = torch.exp2(st['scales'][:, r:r + q.size(0)].t().double() - 128).repeat_interleave(BLOCK, 1)[:, :m]
        total += (q * two).t().contiguous() @ g[r:r + (1 << 19)].double()
    return total
