"""Refusals and host logic of the norm, score and checkpoint operators that an earlier form of them missed; no GPU."""
import pickle

import pytest
import torch


def test_8_bits_are_refused_before_a_forward_whose_gradient_they_cannot_give():
    """A weight whose gradient has more values than a product with a checkpoint gives: said by the forward pass, not by the
    backward pass of an epoch.  With 32 bits, or where the weight needs no gradient, the pass goes on (and may stop here for
    lack of a GPU)."""
    from magnet_amd import MagnetHipError
    from magnet_amd.layer.sparse_magnet import _ChebConvFn
    for k1, cin, cout in ((4, 2048, 2049), (2, 4097, 2048), (1, 1, (1 << 23) + 1)):
        x, w = torch.zeros(1, 2, cin), torch.zeros(1, 1, 1).expand(k1, cin, cout)
        for bits, needs in ((8, True), (32, True), (8, False)):
            said = ''
            try:
                _ChebConvFn.apply(x, w.detach().requires_grad_(needs), None, None, False, None, False, 0, bits)
            except MagnetHipError as e:
                said = str(e)
            except Exception:                          # what a host without a GPU and no Laplacian come to
                pass
            assert ('checkpoint_bits must be 32' in said) == (bits == 8 and needs), (k1, cin, cout, bits, needs, said)


@pytest.mark.parametrize('name', ['ChebNet', 'ChebNet_Edge'])
def test_whole_modules_pickled_before_graph_ptr_still_run(name, monkeypatch):
    """A module object from before the networks had a `graph_ptr` buffer: its trunk is one graph's."""
    from magnet_amd.layer import sparse_magnet
    eye = torch.eye(4).to_sparse()
    net = getattr(sparse_magnet, name)(2, [eye] * 3, [eye] * 3, num_filter=4, K=2, activation=True)
    state = net.__getstate__() if hasattr(net, '__getstate__') else dict(net.__dict__)
    state = dict(state, _buffers={k: v for k, v in net._buffers.items() if k != 'graph_ptr'}, _non_persistent_buffers_set=set())
    old = pickle.loads(pickle.dumps(net))
    old.__dict__.clear()
    old.__setstate__(state)
    monkeypatch.setattr(sparse_magnet, '_run_trunk', lambda *a: a)
    x = torch.zeros(4, 2)
    assert old.trunk(x, x)[3] is None and net.trunk(x, x)[3] is None


def test_sharded_networks_refuse_8_bits_set_after_they_were_made(monkeypatch):
    """checkpoint_bits is an attribute of a convolution and may be set at any time: every pass of a sharded network looks."""
    from magnet_amd import MagnetHipError, dist
    from magnet_amd.layer.sparse_magnet import ChebNet
    eye = torch.eye(4).to_sparse()
    net = ChebNet(2, [eye] * 3, [eye] * 3, num_filter=4, K=2)

    class Part:
        n, rank, world, group, bounds, r0, r1 = 4, 0, 1, None, (0, 4), 0, 4

    for sharded in (dist.ShardedChebNet(net, None, 4, 0, 1), dist.RowShardedChebNet(net, Part())):
        net.Chebs[1].checkpoint_bits = 8
        with pytest.raises(MagnetHipError, match='checkpoint_bits'):
            sharded.trunk(torch.zeros(4, 2, 2))
        net.Chebs[1].checkpoint_bits = 32


@pytest.mark.parametrize('lists', [True, False])
def test_bits_other_than_8_and_32_are_refused_by_every_convolution(lists):
    """Also by one over the reference's lists of matrices, which keeps 32, and by one whose orders the caller keeps."""
    from magnet_amd import MagnetHipError
    from magnet_amd.layer.sparse_magnet import ChebConv
    eye = torch.eye(4).to_sparse()
    conv = ChebConv(2, 4, 2, [eye] * 3, [eye] * 3)
    conv.checkpoint_bits = 16
    if not lists:
        conv._mode, conv.cache_input_propagation = 'cheb', True
    for call in (lambda: conv.forward_packed(torch.zeros(4, 2, 2)), lambda: conv.forward_first(torch.zeros(4, 2), torch.zeros(4, 2))):
        with pytest.raises(MagnetHipError, match='checkpoint_bits' if not lists else 'checkpoint_bits|GPU'):
            call()
    with pytest.raises(MagnetHipError, match='checkpoint_bits'):
        conv.forward_packed(torch.zeros(4, 2, 2))


def test_a_loss_says_what_its_backward_pass_needs():
    """8 bytes a row, and nothing where the backward pass makes maxima and sums again (few classes, class-major, many rows)."""
    import ctypes as C
    from magnet_amd._lib import lib
    size = lib.mh_class_nll_stat_bytes
    assert size(1, 2500, 5, 2500, 1) == 8 * 2500 and size(1, 10 ** 6, 3, 1, 3) == 8 * 10 ** 6 and size(1, 10 ** 6, 40, 10 ** 6, 1) == 8 * 10 ** 6
    assert size(1, 2 * 10 ** 6, 5, 2 * 10 ** 6, 1) == 0 and size(3, 30003, 8, 30003, 1) == 0
    assert size(0, 5, 5, 5, 1) == 0 and size(1, 0, 5, 5, 1) == 0
    fake = C.c_void_p(1 << 20)
    assert lib.mh_class_nll_bwd(fake, 0, 1, 10, 5, 0, 10, 1, fake, -100, None, fake, fake, fake, 0, 10, 1, None) == -1 and b'null' in lib.mh_last_error()


def test_a_checkpoint_without_its_scales_or_gate_is_refused_also_beside_x():
    """codes say that the input is the checkpoint: scales, and the gate of a joined ReLU, are read then, whether X is given or not."""
    import ctypes as C
    from magnet_amd._lib import lib
    fake = C.c_void_p(1 << 20)

    def bwd(x, codes, scales, mask, relu):
        # 4 bytes of workspace: refused for that, and not run, where the pointers are right
        return lib.mh_group_norm_bwd(x, 16, 8, codes, scales, mask, 10, 8, 2, None, 1, fake, None, None, relu, fake, 16, 8, fake, 16, 8,
                                     None, None, fake, 4, None)
    for x in (fake, None):
        for args in ((fake, None, None, 0), (fake, None, fake, 1), (fake, fake, None, 1)):
            assert bwd(x, *args) == -1 and b'null' in lib.mh_last_error(), (x, args)
        assert bwd(x, fake, fake, None, 0) == -4 and bwd(x, fake, fake, fake, 1) == -4
    assert bwd(fake, None, None, None, 1) == -4 and bwd(None, None, None, None, 0) == -1


def test_row_counts_whose_products_leave_64_bits_are_refused():
    """Counts are multiplied by each other and by sizes: beyond 2^40 rows every entry point says so, and a workspace query is 0."""
    import ctypes as C
    from magnet_amd._lib import lib
    fake, top = C.c_void_p(1 << 20), 2 ** 63 - 1
    for n in (2 ** 40 + 1, 2 ** 62, top):
        assert lib.mh_ckpt_store(fake, 8, 4, n, 4, fake, fake, None) == -1 and b'n_rows' in lib.mh_last_error()
        assert lib.mh_ckpt_restore(fake, fake, n, 4, fake, 8, 4, None) == -1 and b'n_rows' in lib.mh_last_error()
        assert lib.mh_ckpt_gram(fake, fake, n, 4, fake, 8, 4, 4, fake, fake, top, None) == -1 and b'n_rows' in lib.mh_last_error()
        assert lib.mh_ckpt_gram_workspace_bytes(n, 4, 4) == 0
    assert 0 < lib.mh_ckpt_gram_workspace_bytes(2 ** 40, 384, 128) < 1 << 30
    for b, n in ((2 ** 32, 2 ** 32), (top, 2), (2, top), (2 ** 21, 2 ** 20), (1, 2 ** 40 + 1)):
        assert lib.mh_class_logprobs(fake, 0, b, n, 5, 0, 1, 5, None, -100, None, fake, None, 0, None, None, 0, 1, 0, None) == -1
        assert b'n_inner' in lib.mh_last_error()
        assert lib.mh_class_nll(fake, 0, b, n, 5, 0, 1, 5, fake, -100, None, fake, fake, fake, fake, 1 << 30, None) == -1
        assert lib.mh_class_nll_bwd(fake, 0, b, n, 5, 0, 1, 5, fake, -100, fake, fake, fake, fake, 0, 1, 5, None) == -1
        assert lib.mh_class_nll_stat_bytes(b, n, 5, 1, 5) == 0
