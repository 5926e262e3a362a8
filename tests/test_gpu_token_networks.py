"""The two ends together, as a program uses them: a network on tokens (embedding, dense layers) whose outputs are trained by the
policy and the preference loss, in SnnNet's flat buffers, eagerly and as one captured step."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
SPECS = [("embed", 41, 9), ("flatten",), ("dense", 54, 32), ("dense", 32, 12)]


def _setup(seed=0, R=48):
    import torch
    from snntc_2023_b200 import nets, train
    net = nets.SnnNet(SPECS, nets.spec_weights(SPECS, 11))
    g = torch.Generator("cuda").manual_seed(seed)
    ids = torch.randint(0, 41, (R, 6), device="cuda", generator=g)
    ids[::5, 4:] = -1                                             # shorter texts
    act = torch.randint(0, 12, (R,), device="cuda", generator=g)
    act[::9] = -1
    adv = torch.randn(R, device="cuda", generator=g)
    starts = torch.tensor([0, 10, 21, 34, R - 2], device="cuda")
    with torch.no_grad():
        lp = train.label_log_probs(net(ids), act)
    return net, ids, act, adv, starts, lp


def _objective(net, ids, act, adv, starts, old, ref):
    from snntc_2023_b200 import train
    out = net(ids)
    return (train.policy_loss(out, act, old, adv, ref_logp=ref, kl_coef=0.2) + 0.5 * train.preference_loss(out, act, starts, beta=0.02)
            + net.constraint_cost(10.0, 1e-3))


def test_gradient_reaches_the_table_through_the_layers():
    """The flat gradient is the layers' own: dX of the first dense layer, summed over each token's places, is the table's. Old
    log-probabilities that differ from the network's, so that the ratio is not one."""
    import torch
    from snntc_2023_b200 import ops
    net, ids, act, adv, starts, lp = _setup()
    old = lp + 0.1 * torch.randn(lp.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    emb = net.layers[0]
    net.flat_grad.fill_(float("nan"))
    net.backward(_objective(net, ids, act, adv, starts, old, lp))
    flat = net.flat_grad.clone()
    assert torch.equal(emb.weight.grad, flat[:41 * 9].view(41, 9)) and emb.grad_sink.data_ptr() == emb.weight.grad.data_ptr()
    # the same objective with the embedding's values as a leaf
    x = ops.snn_embedding(ids, emb.weight.detach(), spikes=True).requires_grad_(True)
    out = x
    for layer in list(net.layers)[1:]:
        out = layer(out)
    from snntc_2023_b200 import train
    rest = (train.policy_loss(out, act, old, adv, ref_logp=lp, kl_coef=0.2) + 0.5 * train.preference_loss(out, act, starts, beta=0.02))
    (dx,) = torch.autograd.grad(rest, x)
    known = ids >= 0
    arg = emb.weight.detach().double()
    sums = torch.zeros(41, 9, dtype=torch.float64, device="cuda").index_put_((ids[known],), dx[known].double(), accumulate=True)
    size = torch.zeros(41, 9, dtype=torch.float64, device="cuda").index_put_((ids[known],), dx[known].double().abs(), accumulate=True)
    n = int(torch.bincount(ids[known]).max())
    assert ((emb.weight.grad.double() - sums * arg.exp()).abs() <= (n + 10) * 2.0 ** -24 * size * arg.exp()).all()
    assert size.sum() > 0


def test_a_captured_training_step_is_the_eager_one():
    import torch
    from snntc_2023_b200 import train
    from snntc_2023_b200.graph import GraphedStep
    finals = []
    for graphed in (False, True):
        net, ids, act, adv, starts, lp = _setup()
        opt = train.Adam(net.flat_param, net.flat_grad, lr=1e-3)

        def step(ids, act, adv, old, ref):
            loss = _objective(net, ids, act, adv, starts, old, ref)
            net.backward(loss)
            opt.step()
            return loss.detach()

        args = (ids, act, adv, lp, lp)
        if graphed:
            run = GraphedStep(step, args, warmup=2)
            for _ in range(4):
                run(*args)
        else:
            for _ in range(6):
                step(*args)
        torch.cuda.synchronize()
        finals.append(net.flat_param.clone())
    assert torch.equal(finals[0], finals[1]) and finals[0].isfinite().all()


def test_texts_through_a_convolution():
    """Ids [B,1,L] are an image one row high: padding tokens never spike, as the padding around it."""
    import torch
    from snntc_2023_b200 import nets
    specs = [("embed", 30, 16), ("conv", 16, 24, 3, 1), ("flatten",), ("dense", 7 * 24, 5)]
    net = nets.SnnNet(specs, nets.spec_weights(specs, 2))
    ids = torch.randint(0, 30, (4, 1, 7), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    short = ids.clone()
    short[:, :, 5:] = -1
    y = net(short)
    assert y.shape == (4, 5)
    loss = net.loss(short, torch.tensor([0, 1, 2, 3], device="cuda"))
    net.backward(loss)
    table = net.layers[0].weight.grad
    assert table.isfinite().all()
    unused = torch.ones(30, dtype=torch.bool, device="cuda")
    unused[short[short >= 0]] = False
    assert (table[unused] == 0).all() and table[~unused].abs().sum() > 0
    with torch.no_grad():
        cut = net.layers[1](net.layers[0](short))[:, :, :4]
        whole = net.layers[1](net.layers[0](short[:, :, :5]))[:, :, :4]
    assert torch.equal(cut, whole)                                # fields that do not reach the padding see none of it


def test_a_capture_beside_a_live_eager_network_is_refused():
    """The loss says so for the leaves behind it, too, not only for its own; and only where the pass gets to them."""
    import torch
    from snntc_2023_b200 import train
    w = torch.randn(6, 5, device="cuda").requires_grad_(True)
    act = torch.tensor([0, 1, -1, 4], device="cuda")
    x, old, adv = torch.randn(4, 6, device="cuda"), torch.full((4,), -1.6, device="cuda"), torch.ones(4, device="cuda")
    alive = train.policy_loss((x @ w).exp(), act, old, adv)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            train.policy_loss((x @ w).exp(), act, old, adv).backward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (x @ w).exp()
        (dout,) = torch.autograd.grad(train.policy_loss(out, act, old, adv), out)
    graph.replay()
    leaf = (x @ w).exp().detach().requires_grad_(True)
    train.policy_loss(leaf, act, old, adv).backward()
    torch.cuda.synchronize()
    assert torch.equal(dout, leaf.grad)
    alive.backward()
    assert w.grad.isfinite().all()
