"""Refusals of the checkpoint, norm and score operators that need no GPU: bad arguments come back as errors of the C ABI or as
MagnetHipError before anything is launched."""
import ctypes as C

import pytest
import torch

FAKE = C.c_void_p(1 << 20)
ODD = C.c_void_p((1 << 20) + 2)


def _lib():
    from magnet_amd import _lib
    return _lib.lib


def _says(lib, rc, code, word):
    assert rc == code and word in lib.mh_last_error(), (rc, lib.mh_last_error())


def test_checkpoint_entry_points_refuse_bad_arguments():
    lib = _lib()
    _says(lib, lib.mh_ckpt_store(FAKE, 8, 4, -1, 4, FAKE, FAKE, None), -1, b'n_rows')
    _says(lib, lib.mh_ckpt_store(FAKE, 8, 4, 5, 0, FAKE, FAKE, None), -1, b'm=0')
    _says(lib, lib.mh_ckpt_store(None, 8, 4, 5, 4, FAKE, FAKE, None), -1, b'null')
    _says(lib, lib.mh_ckpt_store(FAKE, 8, 4, 5, 4, None, FAKE, None), -1, b'null')
    _says(lib, lib.mh_ckpt_store(FAKE, 8, 4, 5, 4, ODD, FAKE, None), -1, b'aligned')
    _says(lib, lib.mh_ckpt_store(FAKE, -8, 4, 5, 4, FAKE, FAKE, None), -1, b'stride')
    _says(lib, lib.mh_ckpt_restore(FAKE, FAKE, 5, 4, FAKE, 3, 4, None), -1, b'stride')
    _says(lib, lib.mh_ckpt_restore(FAKE, FAKE, 5, 4, None, 8, 4, None), -1, b'null')
    _says(lib, lib.mh_ckpt_gram(FAKE, FAKE, 5, 4, FAKE, 8, 4, 0, FAKE, FAKE, 1 << 30, None), -1, b'n=0')
    _says(lib, lib.mh_ckpt_gram(FAKE, FAKE, 5, 4, FAKE, 8, 4, 4, FAKE, FAKE, 16, None), -4, b'workspace')
    _says(lib, lib.mh_ckpt_gram(FAKE, FAKE, 5, 4, None, 8, 4, 4, FAKE, FAKE, 1 << 30, None), -1, b'null')
    _says(lib, lib.mh_ckpt_gram(FAKE, FAKE, 5, 1 << 20, FAKE, 8, 4, 1 << 20, FAKE, FAKE, 1 << 40, None), -1, b'n=')
    assert lib.mh_ckpt_store(None, 0, 0, 0, 4, None, None, None) == 0
    assert lib.mh_ckpt_restore(None, None, 0, 4, None, 8, 4, None) == 0
    assert lib.mh_ckpt_gram_workspace_bytes(0, 4, 4) == 0
    # a partial sum of the whole result for at least one slab; no more than 512 tiles' worth and one for each tile's rounding
    for n, m, k in ((1, 1, 1), (2500, 48, 16), (10 ** 6, 384, 128), (10 ** 7, 1024, 256)):
        b = lib.mh_ckpt_gram_workspace_bytes(n, m, k)
        assert 4 * m * k <= b <= 4 * 256 * 128 * (512 + 2 * (m // 128 + 1) * (k // 32 + 1))


def test_group_norm_entry_points_refuse_bad_arguments():
    lib = _lib()
    big = 1 << 40

    def norm(x=FAKE, ld=16, im=8, n=10, f=8, groups=2, ptr=None, graphs=1, y=FAKE, ldy=16, imy=8, ws=FAKE, ws_bytes=big, stats=FAKE, codes=None):
        return lib.mh_group_norm(x, ld, im, n, f, groups, ptr, graphs, 1e-5, None, None, 0, y, ldy, imy, None, codes, None, stats, ws, ws_bytes, None)

    _says(lib, norm(groups=3), -1, b'divide')
    _says(lib, norm(groups=0), -1, b'divide')
    _says(lib, norm(n=-1), -1, b'n_rows')
    _says(lib, norm(f=0, groups=1), -1, b'F=0')
    _says(lib, norm(graphs=2), -1, b'graph_ptr')
    _says(lib, norm(graphs=0), -1, b'n_graphs')
    _says(lib, norm(x=None), -1, b'null')
    _says(lib, norm(stats=None), -1, b'null')
    _says(lib, norm(ldy=4), -1, b'stride')
    _says(lib, norm(codes=FAKE), -1, b'null')                                      # codes without scales
    _says(lib, norm(ws_bytes=8), -4, b'workspace')
    _says(lib, norm(ws=ODD), -1, b'aligned')
    assert norm(x=None, n=0, y=None, graphs=0, ws=None, stats=None) == 0

    def bwd(x=FAKE, codes=None, scales=None, mask=None, relu=0, g=FAKE, ws_bytes=big, lddx=16):
        return lib.mh_group_norm_bwd(x, 16, 8, codes, scales, mask, 10, 8, 2, None, 1, FAKE, None, None, relu, g, 16, 8, FAKE, lddx, 8,
                                     None, None, FAKE, ws_bytes, None)
    _says(lib, bwd(x=None), -1, b'null')
    _says(lib, bwd(x=None, codes=FAKE), -1, b'null')
    _says(lib, bwd(x=None, codes=FAKE, scales=FAKE, relu=1), -1, b'null')          # the gate is missing
    _says(lib, bwd(g=None), -1, b'null')
    _says(lib, bwd(lddx=4), -1, b'stride')
    _says(lib, bwd(ws_bytes=8), -4, b'workspace')
    assert lib.mh_group_norm_workspace_bytes(10 ** 6, 1, 128, 8) < 64 << 20
    assert lib.mh_group_norm_workspace_bytes(10, 1, 8, 0) == 0


def test_score_entry_points_refuse_bad_arguments():
    lib = _lib()

    def report(dtype=0, b=1, n=10, c=5, sn=5, labels=None, lp=None, ent=FAKE, top=0, tl=None, ti=None, x=FAKE):
        return lib.mh_class_logprobs(x, dtype, b, n, c, 0, 1, sn, labels, -100, lp, ent, None, top, tl, ti, 0, 1, top, None)
    _says(lib, report(dtype=3), -1, b'dtype')
    _says(lib, report(c=0), -1, b'classes')
    _says(lib, report(n=-1), -1, b'n_inner')
    _says(lib, report(sn=-1), -1, b'stride')
    _says(lib, report(x=None), -1, b'null')
    _says(lib, report(ent=None), -1, b'null')
    _says(lib, report(labels=FAKE), -1, b'null')
    _says(lib, report(top=6, tl=FAKE, ti=FAKE), -1, b'top=6')
    _says(lib, report(c=40, top=17, tl=FAKE, ti=FAKE), -1, b'top=17')
    _says(lib, report(top=2, tl=FAKE), -1, b'null')
    assert report(n=0, x=None, ent=None) == 0
    need = lib.mh_class_nll_workspace_bytes()

    def nll(labels=FAKE, loss=FAKE, ws=FAKE, ws_bytes=need):
        return lib.mh_class_nll(FAKE, 0, 1, 10, 5, 0, 1, 5, labels, -100, None, loss, FAKE, FAKE, ws, ws_bytes, None)
    _says(lib, nll(labels=None), -1, b'null')
    _says(lib, nll(loss=None), -1, b'null')
    _says(lib, nll(ws=None), -1, b'null')
    _says(lib, nll(ws_bytes=need - 1), -4, b'workspace')
    rc = lib.mh_class_nll_bwd(FAKE, 0, 1, 10, 5, 0, 1, 5, FAKE, -100, None, FAKE, FAKE, FAKE, 0, 1, 5, None)
    _says(lib, rc, -1, b'null')
    rc = lib.mh_class_logprobs_bwd(FAKE, 0, 1, 10, 5, 0, 1, 5, None, -100, FAKE, FAKE, FAKE, 1, None, 0, 0, None, None, 0, 0, 0, FAKE, 0, 1, 5,
                                   None)
    _says(lib, rc, -1, b'null')                                                    # a gradient of logprob without labels


def test_python_entry_points_refuse_what_they_cannot_take():
    from magnet_amd import MagnetHipError
    from magnet_amd.checkpoint import Checkpoint8
    from magnet_amd.layer.norm import ComplexGroupNorm, complex_group_norm
    from magnet_amd.layer.scores import class_logprobs, class_nll
    x = torch.zeros(3, 2, 8)
    for call in (lambda: Checkpoint8.store(x),                                     # CPU tensors
                 lambda: complex_group_norm(x, 2),
                 lambda: class_logprobs(torch.zeros(3, 4)),
                 lambda: class_nll(torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(MagnetHipError):
            call()
    for call in (lambda: Checkpoint8.store(torch.zeros(3, 8)),
                 lambda: Checkpoint8.store(torch.zeros(3, 1, 8)),
                 lambda: Checkpoint8(torch.zeros(6, 32, dtype=torch.uint8), torch.zeros(1, 8, dtype=torch.uint8), (3, 8)),
                 lambda: Checkpoint8(torch.zeros(6, 32, dtype=torch.uint8), torch.zeros(1, 8, dtype=torch.uint8), (3, 2, 0)),
                 lambda: complex_group_norm(torch.zeros(3, 8), 2),
                 lambda: complex_group_norm(x, 2, checkpoint_bits=16),
                 lambda: complex_group_norm(x, 2, eps=-1.0),
                 lambda: complex_group_norm(x, 2, eps=float('nan')),
                 lambda: complex_group_norm(x, 2, graph_ptr=torch.zeros(2)),
                 lambda: ComplexGroupNorm(3, 8),
                 lambda: ComplexGroupNorm(0, 8),
                 lambda: class_logprobs(torch.zeros(4)),
                 lambda: class_logprobs(torch.zeros(3, 4), torch.zeros(4, dtype=torch.int64)),
                 lambda: class_logprobs(torch.zeros(3, 4), top=5),
                 lambda: class_logprobs(torch.zeros(3, 40), top=17),
                 lambda: class_logprobs(torch.zeros(3, 4), top=-1),
                 lambda: class_nll(torch.zeros(3, 4), None),
                 lambda: class_nll(torch.zeros(1, 4, 3), torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(MagnetHipError):
            call()


def test_networks_check_their_new_arguments():
    """norm_groups has to divide the filters; the state_dict keys of a network without norms are the reference's; sharded
    networks refuse what they do not have."""
    import numpy as np
    import scipy.sparse as sp
    from magnet_amd import MagnetHipError
    from magnet_amd.dist import ShardedChebNet
    from magnet_amd.layer.norm import ComplexGroupNorm
    from magnet_amd.layer.sparse_magnet import ChebConv, ChebNet, ChebNet_Edge, _kept_bits
    eye = torch.eye(4).to_sparse()
    lists = ([eye] * 3, [eye] * 3)
    with pytest.raises(MagnetHipError):
        ChebNet(2, *lists, num_filter=6, norm_groups=4)
    net = ChebNet(2, *lists, num_filter=4, K=2, activation=True, layer=2)
    assert sorted(net.state_dict()) == ['Chebs.0.bias', 'Chebs.0.weight', 'Chebs.2.bias', 'Chebs.2.weight', 'Conv.bias', 'Conv.weight']
    for cls in (ChebNet, ChebNet_Edge):
        net = cls(2, *lists, num_filter=4, K=2, activation=True, layer=2, norm_groups=2, checkpoint_bits=8)
        kinds = [type(m).__name__ for m in net.Chebs]
        assert kinds == ['ChebConv', 'ComplexGroupNorm', 'complex_relu_layer'] * 2
        assert all(m.checkpoint_bits == 8 for m in net.Chebs if isinstance(m, (ChebConv, ComplexGroupNorm)))
    assert ChebConv.checkpoint_bits == 32
    with pytest.raises(MagnetHipError):
        _kept_bits(16)
    with torch.no_grad():
        assert _kept_bits(8) == 32                     # nothing is kept where nothing will be differentiated
    assert _kept_bits(8) == 8
    op = sp.csr_matrix(np.eye(4))
    with pytest.raises(MagnetHipError, match='norm'):
        ShardedChebNet(net, op, 4, 0, 1)
    net = ChebNet(2, *lists, num_filter=4, K=2, checkpoint_bits=8)
    with pytest.raises(MagnetHipError, match='checkpoint_bits'):
        ShardedChebNet(net, op, 4, 0, 1)


def test_fused_loss_takes_no_other_criterion():
    from magnet_amd.train import _check_fused
    _check_fused(True, None)
    _check_fused(True, torch.nn.NLLLoss())
    _check_fused(False, torch.nn.MSELoss())
    for c in (torch.nn.MSELoss(), torch.nn.NLLLoss(reduction='sum'), torch.nn.NLLLoss(weight=torch.ones(3)), torch.nn.NLLLoss(ignore_index=0)):
        with pytest.raises(ValueError):
            _check_fused(True, c)


def test_sizes_beyond_the_limits():
    """Workspace queries and entry points at the ends of their types: 0 and an error, no overflow and no division by its result."""
    lib = _lib()
    top = 2 ** 31 - 1
    for m in (1 << 23, 1 << 24, top):
        for n in (1 << 23, 1 << 24, top):
            assert lib.mh_ckpt_gram_workspace_bytes(5, m, n) == 0
    assert lib.mh_ckpt_gram_workspace_bytes(5, 1 << 12, 1 << 12) > 0
    _says(lib, lib.mh_ckpt_gram(FAKE, FAKE, 5, 1 << 24, FAKE, 8, 4, 1 << 24, FAKE, FAKE, 1 << 40, None), -1, b'n=')
    for n, graphs, f in ((2 ** 62, 1, 8), (10, top, 8), (10, 1, top), (10, 1, top - 1)):
        assert lib.mh_group_norm_workspace_bytes(n, graphs, f, 1) == 0
    _says(lib, lib.mh_class_logprobs(FAKE, 0, 1, 10, top, 0, 1, 5, None, -100, None, FAKE, None, 0, None, None, 0, 1, 0, None), -1, b'classes')


def test_drivers_refuse_bad_arguments_at_once():
    from magnet_amd import Edge_sparseMagnet, sparse_Magnet
    for driver in (sparse_Magnet, Edge_sparseMagnet):
        for bad in (['--report', '-1'], ['--norm_groups', '-2'], ['--norm_groups', '3', '--num_filter', '8'], ['--checkpoint_bits', '4']):
            with pytest.raises(SystemExit):
                driver.parse_args(bad)
        assert driver.parse_args(['--report', '2', '--norm_groups', '4', '--num_filter', '8']).report == 2


def test_kept_forward_pass_belongs_to_its_graphs():
    """SharedForwardEpochs: another graph_ptr, or the same one written in place, makes a new pass."""
    from magnet_amd.train import SharedForwardEpochs

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.ones(()))
            self.register_buffer('graph_ptr', torch.tensor([0, 4, 8]), persistent=False)
            self.passes = 0

        def trunk(self, real, imag):
            self.passes += 1
            return self.w * real * float(self.graph_ptr[1])

        def head(self, p):
            return torch.log_softmax(p.t().unsqueeze(0), 1)
    net = Net()
    epochs = SharedForwardEpochs(net, torch.optim.SGD(net.parameters(), lr=0.1))
    x, label, index = torch.randn(8, 3), torch.zeros(1, 8, dtype=torch.int64), torch.arange(8)
    run = lambda: epochs.node_epoch(x, x, label, index, index)
    run()
    assert net.passes == 2
    run()
    assert net.passes == 3                                         # the evaluation's only
    net.graph_ptr[1] = 2
    run()
    assert net.passes == 5
    net.graph_ptr = torch.tensor([0, 2, 8])
    run()
    assert net.passes == 7
    run()
    assert net.passes == 8
