"""CPU-side checks of the two ends of a network on tokens: status codes before anything touches a device, refusals of the
Python entry points, the embedding layer's surface, its place in networks and checkpoints."""
import numpy as np
import pytest
import torch

FAKE = 0x1000      # never dereferenced: every call below is rejected during validation


def test_status_codes_of_the_embedding():
    from snntc_2023_b200 import _lib
    lib = _lib.load()
    fwd = lambda ids=FAKE, b=8, table=FAKE, y=FAKE, N=5, V=7, D=3: lib.snntc_embedding_forward(ids, b, table, y, N, V, D, 1.0, 0, -1, 1e5, 0)  # noqa: E731
    assert fwd(ids=0) == fwd(table=0) == fwd(y=0) == -1
    assert fwd(N=-1) == fwd(V=0) == fwd(D=0) == -2
    assert fwd(N=1 << 31) == fwd(V=(1 << 31) - 1) == fwd(D=(1 << 30) + 1) == -4
    assert fwd(b=2) == -8
    assert fwd(N=0, ids=0, table=0, y=0) == 0
    size = lib.snntc_embedding_backward_workspace_bytes
    assert size(0, 7, 3) == 0 and size(1000, 7, 3) >= 2 * 1000 * 8
    bwd = lambda ids=FAKE, g=FAKE, table=0, dt=FAKE, N=5, V=7, D=3, spikes=0, ws=FAKE, n=1 << 40: lib.snntc_embedding_backward(  # noqa: E731
        ids, 8, 0, g, table, dt, N, V, D, 1.0, spikes, -1, ws, n, 0)
    assert bwd(ids=0) == bwd(g=0) == bwd(dt=0) == bwd(spikes=1) == -1
    assert bwd(N=-1) == bwd(V=0) == bwd(D=0) == -2
    assert bwd(ws=0) == bwd(ws=FAKE + 8) == bwd(n=size(5, 7, 3) - 1) == -5
    kept, scratch = lib.snntc_embedding_sorted_bytes, lib.snntc_embedding_sort_workspace_bytes
    assert kept(0, 9) == kept(8192, 9999) == scratch(8192, 9999) == kept(8193, 9) == 0   # a short lookup: the backward sorts
    assert kept(8193, 512) == 8193 * 8 and scratch(8193, 512) > 8193 * 8
    both = lambda ids=FAKE, table=FAKE, y=FAKE, out=FAKE, N=9000, ws=FAKE, n=1 << 40: lib.snntc_embedding_forward_sort(  # noqa: E731
        ids, 8, table, y, N, 7, 512, 1.0, 0, -1, 1e5, out, ws, n, 0)
    assert both(ids=0) == both(table=0) == both(y=0) == both(out=0) == -1
    assert both(ws=0) == both(ws=FAKE + 8) == both(out=FAKE + 8) == both(n=scratch(9000, 512) - 1) == -5
    assert both(N=0, ids=0, table=0, y=0, out=0, ws=0) == 0


def test_status_codes_of_the_losses_on_choices():
    from snntc_2023_b200 import _lib
    lib = _lib.load()
    lp = lambda z=FAKE, lab=FAKE, out=FAKE, R=4, J=3: lib.snntc_label_logp_forward(z, lab, out, 0, R, J, 0)  # noqa: E731
    assert lp(z=0) == lp(lab=0) == lp(out=0) == -1
    assert lp(R=0) == lp(J=0) == lp(R=-1) == -2
    assert lp(R=1 << 31) == lp(J=(1 << 30) + 1) == -4
    args = [FAKE] * 6
    for k in (0, 1, 2, 3, 5):
        a = list(args)
        a[k] = 0
        assert lib.snntc_choice_backward(*a, 4, 3, 0) == -1
    assert lib.snntc_choice_backward(*args, 0, 3, 0) == -2
    assert lib.snntc_scale_gradient(0, FAKE, 4, 0) == lib.snntc_scale_gradient(FAKE, 0, 4, 0) == -1
    assert lib.snntc_scale_gradient(FAKE, FAKE, 0, 0) == 0
    pol = lambda p=(FAKE,) * 10, R=4, J=3, lo=0.2, hi=0.2, kl=0.1, ws=FAKE, n=1 << 40: lib.snntc_policy_loss(*p, R, J, lo, hi, kl, ws, n, 0)  # noqa: E731
    for k in (0, 1, 2, 3, 5, 6):
        p = [FAKE] * 10
        p[k] = 0
        assert pol(p) == -1
    assert pol(R=0) == pol(J=0) == -2
    assert pol(lo=-0.1) == pol(lo=1.1) == pol(hi=-0.1) == pol(lo=float("nan")) == pol(kl=float("inf")) == -8
    assert pol([FAKE] * 4 + [0] + [FAKE] * 5) == -8                          # a KL term without a reference
    assert pol(ws=0) == pol(ws=FAKE + 8) == pol(n=lib.snntc_policy_loss_workspace_bytes(4) - 1) == -5
    pre = lambda p=(FAKE,) * 8, R=8, J=3, P=2, beta=0.1, eps=0.0, ws=FAKE, n=1 << 40: lib.snntc_preference_loss(*p, R, J, P, beta, eps, ws, n, 0)  # noqa: E731
    for k in (0, 1, 4, 5, 6, 7):
        p = [FAKE] * 8
        p[k] = 0
        assert pre(p) == -1
    assert pre(P=0) == pre([FAKE, FAKE, 0] + [FAKE] * 5, P=3) == -2          # eight rows are no six equal texts
    assert pre(beta=float("nan")) == pre(eps=-0.1) == pre(eps=1.5) == -8
    assert pre(ws=0) == pre(ws=FAKE + 8) == pre(n=lib.snntc_preference_loss_workspace_bytes(8, 2) - 1) == -5


def test_entry_points_refuse_cpu_tensors():
    from snntc_2023_b200 import _lib, ops, train
    z, lab = torch.ones(4, 3), torch.zeros(4, dtype=torch.long)
    for call in (lambda: ops.snn_embedding(lab, z), lambda: train.label_log_probs(z, lab),
                 lambda: train.policy_loss(z, lab, torch.zeros(4), torch.zeros(4)),
                 lambda: train.preference_loss(z, lab, torch.tensor([0, 2, 4]))):
        with pytest.raises(_lib.SnntcError, match="no CPU implementation"):
            call()


def test_embedding_layer_surface():
    import SNN_TC_Modules as SNN
    e = SNN.SNN_embedding(11, 6)
    assert tuple(e.weight.shape) == (11, 6) and e.weight.dtype == torch.float32 and e.weight.requires_grad
    assert 0 <= float(e.weight.min()) and float(e.weight.max()) < 1 and e.spikes and e.grad_sink is None and callable(e.call)
    assert np.allclose(SNN.SNN_embedding(2, 3, weight=np.arange(6).reshape(2, 3)).weight.detach().numpy(), np.arange(6).reshape(2, 3))
    with pytest.raises(ValueError):
        SNN.SNN_embedding(2, 3, weight=np.zeros((3, 2)))


def test_networks_on_tokens_are_stored_and_named(tmp_path):
    from snntc_2023_b200 import checkpoint, nets
    specs = [("embed", 7, 5), ("flatten",), ("dense", 15, 4)]
    ws = nets.spec_weights(specs, 3)
    assert [w.shape for w in ws] == [(7, 5), (16, 4)] and ws[0].min() >= 0 and ws[0].max() < 1
    net = nets.SnnNet(specs, ws, device="cpu")
    emb, dense = net.parameter_layers()
    assert net.weighted_layers() == [dense]                       # no part of the constraint cost
    assert net.flat_param.numel() == 36 + 64                      # 35 weights of the table, the next ones on 16 bytes again
    assert dense.weight.data_ptr() == net.flat_param.data_ptr() + 36 * 4 and float(net.flat_param[35]) == 0.0
    assert emb.grad_sink.data_ptr() == net.flat_grad.data_ptr() and emb.grad_sink.shape == emb.weight.shape
    rows = nets.layer_work(specs, (3,))
    assert rows == [dict(kind="dense", R=1, I=16, J=4, needs_dx=True)]
    conv = nets.layer_work([("embed", 7, 5), ("conv", 5, 8, 3, 1)], (1, 6))
    assert conv == [dict(kind="conv", R=6, I=46, J=8, needs_dx=True)]
    names = [n for n, _ in checkpoint.keras_names(net)]
    assert names == ["snn_embedding/embkernel:0", "snn_dense/fckernel:0"]
    path = str(tmp_path / "w.npz")
    checkpoint.save_weights(net, path)
    other = nets.SnnNet(specs, nets.spec_weights(specs, 4), device="cpu")
    checkpoint.load_weights(other, path)
    assert torch.equal(other.flat_param, net.flat_param)
