#!/usr/bin/env python3
"""Times and kernels of the cases of perf/operators.py (checkpoints in 8 bits, group norm, class scores), and training epochs with them.

    python3 tools/operators_profile.py time [CASE ...]        whole passes of the plain form and of the kernels, in turn, and
                                                              the error of either against 64 bits
    rocprofv3 --kernel-trace --output-format csv -d DIR/CASE -- python3 tools/operators_profile.py run CASE
    python3 tools/operators_profile.py kernels DIR            median time of every kernel of a pass, for each DIR/CASE
    python3 tools/operators_profile.py sweep                  widths and batches beside the cases, as replayed graphs
    python3 tools/operators_profile.py epochs                 epochs at 2M nodes with and without 8 bits, norms, fused loss

profiles/operators_kernels.txt is the output of `time`, `kernels` and `sweep`, profiles/operators_epochs.txt that of `epochs`."""
import collections
import csv
import glob
import os
import re
import statistics
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
PASSES = 9


def cases(names):
    from perf import operators
    listed = operators.listed()
    return operators, [c for c in listed if not names or c['name'] in names]


def norm(t):
    return float(t.double().norm())


def error(outs, exact):
    """Largest relative error in norm over the outputs that are computed numbers."""
    outs, exact = [list(v) if isinstance(v, (list, tuple)) else [v] for v in (outs, exact)]
    return max(norm(o.to(e.device).double() - e) / max(norm(e), 1e-300) for o, e in zip(outs, exact) if e is not None and o.is_floating_point())


def definition(P, case, seed):
    """64 bits; a norm of a moderate size on the host: torch's means over two dimensions vary on the GPU."""
    if case['op'] == 'norm' and case['nodes'] * case['feats'] <= 2e7:
        st = P.prepare(case, seed)
        return P._exact_norm(case, {k: v.cpu() if hasattr(v, 'cpu') else v for k, v in st.items()})
    return P.exact(case, seed)


def passes(names):
    import torch
    P, todo = cases(names)
    for case in todo:
        times = {False: [], True: []}
        states = [P.prepare(case, k) for k in (1, 2, 3)]
        for turn in range(4):
            for own in (False, True):
                P.own = own
                for st in states:
                    P.run(st)
                torch.cuda.synchronize()
                n = 6
                t = time.perf_counter()
                while True:
                    for k in range(n):
                        P.run(states[k % 3])
                    torch.cuda.synchronize()
                    spent = time.perf_counter() - t
                    if spent > 0.1:
                        break
                    n, t = 4 * n, time.perf_counter()
                times[own].append(spent / n * 1e6)
        plain, here = min(times[False]), min(times[True])
        print('%-20s plain form %10.2f us   kernels %10.2f us   %.2fx' % (case['name'], plain, here, plain / here), flush=True)
        e, errors = definition(P, case, 1), []
        for own in (False, True):
            P.own = own
            errors.append(error(P.run(states[0]), e))
        print('%-20s error      %10.2g      kernels %10.2g' % (case['name'], *errors), flush=True)


def run(name):
    import torch
    P, todo = cases([name])
    P.own = True
    states = [P.prepare(todo[0], k) for k in (1, 2, 3)]
    for k in range(PASSES):
        P.run(states[k % 3])
    torch.cuda.synchronize()
    print('done', name, flush=True)


def kernels(top):
    for case in cases([])[1]:
        found = glob.glob(os.path.join(top, case['name'], '**', '*kernel_trace.csv'), recursive=True)
        if not found:
            continue
        spent = collections.defaultdict(list)
        for row in csv.DictReader(open(found[0])):
            if re.search(r'ckpt_|norm_\w*kernel|score_|nll_', row['Kernel_Name']):
                spent[row['Kernel_Name']].append((int(row['End_Timestamp']) - int(row['Start_Timestamp'])) / 1e3)
        print(case['name'])
        total = 0.0
        for kernel, v in sorted(spent.items(), key=lambda kv: -sum(kv[1])):
            total += statistics.median(v) * len(v) / PASSES
            print('%9.2f us  %s' % (statistics.median(v), kernel.replace('void ', '').replace('(anonymous namespace)::', '')[:60]))
        print('%9.2f us total per pass' % total)


def replayed(f, n):
    """Best time of a pass, us, of 5 runs of n replays."""
    import torch
    f()
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    best = float('inf')
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            graph.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) / n * 1e3)
    return best


def sweep():
    import torch
    from magnet_amd._lib import lib
    from magnet_amd.checkpoint import Checkpoint8
    from magnet_amd.layer.norm import complex_group_norm
    from magnet_amd.layer.scores import class_logprobs, class_nll
    for m, k in ((384, 128), (416, 128), (512, 128), (512, 96), (768, 128)):
        ck, g = Checkpoint8.store(torch.randn(1_000_000, 2, m, device='cuda')), torch.randn(1_000_000, 2, k, device='cuda')
        print('gram 1M x %d x %d: %.0f us' % (m, k, replayed(lambda: ck.gram(g), 10)), flush=True)
    grad = torch.autograd.grad
    for dtype in (torch.float32, torch.bfloat16):
        for rows, c, layout in [(60001, c, 'row') for c in (65, 100, 128, 172, 349, 500, 1000)] + [(1_000_000, 3, 'row'), (2_000_000, 40, 'class'), (200_000, 40, 'class')]:
            s = (3 * torch.randn((1, c, rows) if layout == 'class' else (rows, c), device='cuda')).to(dtype)
            lab = torch.randint(0, c, (1, rows) if layout == 'class' else (rows,), device='cuda')
            gl, gh, one = torch.randn(lab.shape, device='cuda'), torch.randn(lab.shape, device='cuda'), torch.ones((), device='cuda')

            def loss():
                x = s.detach().requires_grad_()
                return grad(class_nll(x, lab)[0], x, one)

            def report():
                x = s.detach().requires_grad_()
                r = class_logprobs(x, lab, top=min(5, c))
                return grad([r.logprob, r.entropy], x, [gl, gh])
            t = [replayed(f, 20) for f in (lambda: class_nll(s, lab), loss, lambda: class_logprobs(s, lab, top=min(5, c)), report)]
            print('%8d x %4d %5s %s  read at the copy rate %.1f | loss %.1f, its gradient %.1f | report of 5 %.1f, its gradient %.1f us'
                  % (rows, c, layout, str(dtype)[6:], s.numel() * s.element_size() / 4.7e6, t[0], t[1] - t[0], t[2], t[3] - t[2]), flush=True)
    n, f, groups = 1_000_000, 64, 8
    x, g, w, b = torch.randn(n, 2, f, device='cuda'), torch.randn(n, 2, f, device='cuda'), torch.ones(f, device='cuda'), torch.zeros(f, device='cuda')
    for graphs in (1, 512, 2000, 10000, 50000, 200000):
        inner = torch.sort(torch.randint(0, n + 1, (graphs - 1,), device='cuda'))[0].int()
        ptr = torch.nn.functional.pad(torch.nn.functional.pad(inner, (1, 0)), (0, 1), value=n)

        def train():
            leaves = [v.detach().requires_grad_() for v in (x, w, b)]
            return grad(complex_group_norm(leaves[0], groups, *leaves[1:], graph_ptr=ptr, relu=True), leaves, g)
        t = replayed(lambda: complex_group_norm(x, groups, w, b, graph_ptr=ptr, relu=True), 5)
        print('norm 1M x 64, %d graphs: forward %.0f, backward %.0f us, workspace %.0f MB (input 512)'
              % (graphs, t, replayed(train, 5) - t, lib.mh_group_norm_workspace_bytes(n, graphs, f, groups) / 1e6), flush=True)


def epochs():
    import torch
    from magnet_amd.laplacian import build_magnetic_laplacian, powerlaw_edges
    from magnet_amd.layer.sparse_magnet import ChebNet
    from magnet_amd.train import NodeTargets, node_epoch
    from magnet_amd.utils.hermitian import ChebBasis
    n, f, k = 2_000_000, 128, 2
    src, dst = powerlaw_edges(n, 40_000_000, 43, device='cuda')
    lap = build_magnetic_laplacian(src, dst, n, q=0.25)
    del src, dst
    x, lab, idx = torch.randn(n, f, device='cuda'), torch.randint(0, 5, (1, n), device='cuda'), torch.randperm(n, device='cuda')
    train, val = NodeTargets(lab, idx[:n // 2]), NodeTargets(lab, idx[n // 2:])
    print('ChebNet training epochs (forward, backward, Adam, evaluation forward), one MI355X, power-law digraph of 40M edges.')
    print('nodes, filters, K, convolutions, options, time of an epoch, peak memory above what lives between epochs, loss after 7 epochs')
    bits, norms = dict(checkpoint_bits=8), dict(norm_groups=8)
    for layer, options in ((2, (({}, False), ({}, True), (bits, False), (bits, True), (norms, True), ({**norms, **bits}, True))),
                           (4, (({}, True), (bits, True), (norms, True), ({**norms, **bits}, True)))):
        for kw, fused in options:
            torch.manual_seed(0)
            torch.cuda.empty_cache()
            net = ChebNet(f, ChebBasis(lap, k), None, num_filter=f, K=k, label_dim=5, activation=True, layer=layer, **kw).to('cuda')
            opt = torch.optim.Adam(net.parameters(), lr=1e-3)
            for _ in range(2):
                node_epoch(net, opt, x, x, lab, train, val, fused_loss=fused)
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            base, t = torch.cuda.memory_allocated(), time.perf_counter()
            for _ in range(5):
                r = node_epoch(net, opt, x, x, lab, train, val, fused_loss=fused)
            torch.cuda.synchronize()
            ms = (time.perf_counter() - t) / 5 * 1e3
            print(n, f, k, layer, kw, 'fused' if fused else '', '%.1f ms  peak %.1f GB above %.1f GB  loss %.5f'
                  % (ms, (torch.cuda.max_memory_allocated() - base) / 1e9, base / 1e9, float(r[0])), flush=True)
            del net, opt, r


if __name__ == '__main__':
    what, rest = sys.argv[1], sys.argv[2:]
    {'time': lambda: passes(rest), 'run': lambda: run(rest[0]), 'kernels': lambda: kernels(rest[0]), 'sweep': sweep, 'epochs': epochs}[what]()
