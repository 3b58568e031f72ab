"""GPU: ModelBiLSTM in training (models.py train(), training.py): logits and all gradients of the whole model against the same
graph in 64 bits on the CPU, the reference's training step (cross entropy with class weights, clipping, optimizer) run with the
library's operators, the trained values in the inference kernels, and steps captured into HIP graphs."""
import math

import numpy as np
import pytest
import torch

from oracle import forward_np as onp

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24


def build(**kw):
    from deepsignal_plant_amd.models import ModelBiLSTM
    cfg = onp.OracleConfig(**kw)
    m = ModelBiLSTM(cfg.seq_len, cfg.signal_len, cfg.num_layers1, cfg.num_layers2, cfg.num_classes, 0.0, cfg.hidden_size, cfg.vocab_size,
                    cfg.embedding_size, cfg.is_base, cfg.is_signallen, module=cfg.module, device=0, init_state="zeros")
    w = onp.make_weights(cfg, 11, 1.5)
    m.load_state_dict({k: torch.from_numpy(v) for k, v in w.items()})
    return cfg, m, w


def plain(cfg, p, ins, states):
    """models.py:178-240 on torch tensors of any type: the arithmetic of the oracle's forward, differentiable"""
    kmer, means, stds, lens, signals = ins
    n, L, H = kmer.shape[0], cfg.seq_len, cfg.hidden_size

    def bilstm(x, prefix, layers, h0, c0):
        for k in range(layers):
            out = []
            for d, way in enumerate(("", "_reverse")):
                w_ih, w_hh, b_ih, b_hh = (p["%s.%s_l%d%s" % (prefix, a, k, way)] for a in ("weight_ih", "weight_hh", "bias_ih", "bias_hh"))
                h, c, ys = h0[2 * k + d], c0[2 * k + d], [None] * L
                for t in range(L)[::-1 if d else 1]:
                    i, f, g, o = (x[:, t] @ w_ih.t() + b_ih + h @ w_hh.t() + b_hh).chunk(4, 1)
                    c = f.sigmoid() * c + i.sigmoid() * g.tanh()
                    h = o.sigmoid() * c.tanh()
                    ys[t] = h
                out.append(torch.stack(ys, 1))
            x = torch.cat(out, 2)
        return x
    parts = []
    if cfg.module != "signal_bilstm":
        x = [means[..., None], stds[..., None]]
        if cfg.is_base:
            x.insert(0, p["embed.weight"][kmer.long()])
        if cfg.is_signallen:
            x.append(lens[..., None])
        x = bilstm(torch.cat(x, 2), "lstm_seq", cfg.num_layers2, states["h_seq"], states["c_seq"])
        parts.append(torch.relu(x @ p["fc_seq.weight"].t() + p["fc_seq.bias"]))
    if cfg.module != "seq_bilstm":
        x = bilstm(signals, "lstm_signal", cfg.num_layers2, states["h_sig"], states["c_sig"])
        parts.append(torch.relu(x @ p["fc_signal.weight"].t() + p["fc_signal.bias"]))
    x = bilstm(torch.cat(parts, 2), "lstm_comb", cfg.num_layers1, states["h_comb"], states["c_comb"])
    x = torch.relu(torch.cat((x[:, -1, :H], x[:, 0, H:]), 1) @ p["fc1.weight"].t() + p["fc1.bias"])
    return x @ p["fc2.weight"].t() + p["fc2.bias"]


def batch(cfg, n, seed=5):
    ins = [torch.from_numpy(a) for a in onp.make_inputs(cfg, n, seed)]
    labels = torch.randint(0, cfg.num_classes, (n,), generator=torch.Generator().manual_seed(seed))
    return ins, labels


CONFIGS = [dict(), dict(module="seq_bilstm", num_layers1=2, hidden_size=64), dict(module="signal_bilstm", hidden_size=100, num_layers1=1),
           dict(hidden_size=40, num_layers2=2, is_base=False, num_classes=3), dict(hidden_size=136, is_signallen=False, seq_len=9, signal_len=12)]


@pytest.mark.parametrize("kw", CONFIGS)
def test_model_gradients_against_64_bits(kw):
    """every parameter's gradient, through all layers.  Each layer's products are off by n U of their sizes (n: their length) and hand
    that on: 2 passes x 13 steps x 6 layers of products of up to 1,024 -- by the norm, and with the errors' signs mixed, below
    their root: 2 * 13 * 6 * 1,024 ** 0.5 * U = 3e-4"""
    from deepsignal_plant_amd import train_ops as ops
    cfg, m, w = build(**kw)
    n = 70
    ins, labels = batch(cfg, n)
    states = onp.make_init_states(cfg, n, 4)
    weight = torch.linspace(1.0, 1.8, cfg.num_classes)
    m.train()
    logits, probs = m(*[t.to(DEV) for t in ins], init_states={k: torch.from_numpy(v) for k, v in states.items()})
    loss = ops.cross_entropy(logits, labels.to(DEV), weight=weight.to(DEV))
    loss.backward()
    p = {k: torch.from_numpy(v).double().requires_grad_() for k, v in w.items()}
    want = plain(cfg, p, [t.double() for t in ins], {k: torch.from_numpy(v).double() for k, v in states.items()})
    lp = torch.log_softmax(want, 1)
    wl = weight.double()[labels]
    (-(lp.gather(1, labels[:, None])[:, 0] * wl).sum() / wl.sum()).backward()
    tol = 2 * 13 * 6 * 1024 ** 0.5 * U
    assert (logits.detach().double().cpu() - want.detach()).norm() <= tol * want.detach().norm()
    assert (probs.detach().double().cpu() - lp.detach().exp()).abs().max() <= tol
    assert [k for k, _ in m.named_parameters()] == list(p)
    for k, v in m.named_parameters():
        if p[k].grad is None:   # an embedding that the model does not use
            assert v.grad is None and k == "embed.weight" and not cfg.is_base
            continue
        off = float((v.grad.double().cpu() - p[k].grad).norm())
        assert off <= tol * float(p[k].grad.norm()) + 1e-12, (k, off / float(p[k].grad.norm()))
    # the clipping of the whole model, as the reference has it
    norm = float(ops.clip_grad_norm_(m.parameters(), 0.05))
    total = math.sqrt(sum(float((v.grad ** 2).sum()) for v in p.values() if v.grad is not None))
    assert abs(norm - total) <= tol * total
    after = math.sqrt(sum(float((v.grad.double() ** 2).sum()) for v in m.parameters() if v.grad is not None))
    assert abs(after - min(total, 0.05)) <= 2e-4 * min(total, 0.05)


def test_training_forward_equals_the_inference_kernels():
    cfg, m, w = build(hidden_size=96)
    ins, _ = batch(cfg, 300)
    dev = [t.to(DEV) for t in ins]
    states = {k: torch.from_numpy(v) for k, v in onp.make_init_states(cfg, 300, 4).items()}
    logits, probs = m.cuda(0).eval()(*dev, init_states=states)
    tl, tp, lab = m.train()(*dev, init_states=states, want_labels=True)
    assert (probs - tp.detach()).abs().max() < 1e-5 and (logits - tl.detach()).abs().max() < 1e-4
    assert torch.equal(lab, tp.argmax(1).to(torch.uint8))
    zl, _ = m(*dev)
    ez, _ = m.eval()(*dev)
    assert (zl.detach() - ez).abs().max() < 1e-4
    with pytest.raises(ValueError, match="site_keys"):
        m.train()(*dev, site_keys=torch.arange(300, device=DEV))
    with pytest.raises(RuntimeError, match="must live on"):
        m(*ins)
    with pytest.raises(ValueError, match="initial state"):
        m(*dev, init_states={"h_comb": torch.zeros(1, 2, 3)})


def step_of(m, ops, opt, dev, labels, weight):
    opt.zero_grad()
    logits, _ = m(*dev)
    loss = ops.cross_entropy(logits, labels, weight=weight)
    loss.backward()
    norm = ops.clip_grad_norm_(m.parameters(), 0.5)
    opt.step()
    return loss.detach(), norm


def test_a_training_loop_and_what_the_inference_kernels_get():
    """optimizer steps as train.py:104-128 takes them; the parameters stay the same tensors, a checkpoint round-trips, and eval() serves
    the trained values"""
    from deepsignal_plant_amd import train_ops as ops
    cfg, m, w = build(hidden_size=48, num_layers1=2)
    m.dropout_rate = 0.5
    m.init_state = "randn"
    ins, labels = batch(cfg, 512)
    dev, y, weight = [t.to(DEV) for t in ins], labels.to(DEV), torch.tensor([1.0, 1.5], device=DEV)
    before = m.cuda(0).eval()(*dev)[1].clone()
    opt = torch.optim.Adam(m.parameters(), lr=1e-3)
    m.train()
    ids = [id(v) for v in m.parameters()]
    for _ in range(3):
        loss, norm = step_of(m, ops, opt, dev, y, weight)
        assert math.isfinite(float(loss)) and float(norm) > 0
    assert [id(v) for v in m.parameters()] == ids
    sd = m.state_dict()
    assert all(torch.equal(sd[k], v.detach().cpu()) for k, v in m.named_parameters())
    assert any(not np.array_equal(sd[k].numpy(), w[k]) for k in w)
    m.init_state = "zeros"
    m.dropout_rate = 0.0
    trained = m(*dev)[1].detach()
    served = m.eval()(*dev)[1]
    assert (served - trained).abs().max() < 1e-5 and (served - before).abs().max() > 1e-5
    cfg2, other, _ = build(hidden_size=48, num_layers1=2)
    other.load_state_dict(sd)
    assert torch.equal(other.cuda(0).eval()(*dev)[1], served)
    m.load_state_dict({k: torch.from_numpy(v) for k, v in w.items()})   # into the leaves too
    assert all(np.array_equal(v.detach().cpu().numpy(), w[k]) for k, v in m.named_parameters())
    m.train()
    m.zero_grad()
    assert all(v.grad is None for v in m.parameters())


def test_inference_sees_what_is_written_to_the_parameters():
    """an optimizer step after eval(), a value written by hand, and a partial state_dict over trained values"""
    from deepsignal_plant_amd import train_ops as ops
    cfg, m, w = build(hidden_size=48, num_layers1=2)
    ins, labels = batch(cfg, 64)
    dev = [t.to(DEV) for t in ins]
    m.cuda(0).train()
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    ops.cross_entropy(m(*dev)[0], labels.to(DEV)).backward()
    m.eval()
    before = m(*dev)[0].clone()
    opt.step()
    after = m(*dev)[0].clone()
    assert (after - before).abs().max() > 1e-4 and torch.equal(m(*dev)[0], after)
    leaves = dict(m.named_parameters())
    with torch.no_grad():
        leaves["fc2.bias"].add_(1.0)
    assert (m(*dev)[0] - after - 1.0).abs().max() < 1e-5
    trained = leaves["fc1.weight"].detach().clone()
    m.load_state_dict({"fc2.bias": torch.from_numpy(w["fc2.bias"])}, strict=False)
    assert torch.equal(leaves["fc1.weight"], trained) and torch.equal(m.state_dict()["fc1.weight"], trained.cpu())
    assert np.array_equal(leaves["fc2.bias"].detach().cpu().numpy(), w["fc2.bias"])
    kmer, rest = dev[0], dev[1:]
    m.train()
    want = m(*dev)[0].detach()
    for t in (torch.float64, torch.int16, torch.int64, torch.uint8):
        assert torch.equal(m(kmer.to(t), *rest)[0].detach(), want)


def test_inference_sees_writes_that_leave_no_mark_on_the_parameters():
    """after eval(): values copied through .data, another tensor put there, a vector of parameters, a fused optimizer's step, the
    replay of a captured step: none moves a tensor's version, and the next inference call computes with what they wrote"""
    cfg, m, _ = build(hidden_size=48, num_layers1=1)
    ins, _ = batch(cfg, 64)
    dev = [t.to(DEV) for t in ins]
    m.cuda(0).train()
    params = m.parameters()
    for p in params:
        p.grad = torch.full_like(p, 0.01)
    m.eval()

    def served(what):
        _, other, _ = build(hidden_size=48, num_layers1=1)
        other.load_state_dict({k: v.detach().cpu() for k, v in m.named_parameters()})
        want = other.cuda(0).eval()(*dev)[0]
        got = m(*dev)[0].clone()
        assert torch.equal(got, want), what
        assert all(torch.equal(v, p.detach().cpu()) for v, p in zip(m.state_dict().values(), params)), what
        return got
    before = served("nothing written")

    def moved(what):
        nonlocal before
        now = served(what)
        assert not torch.equal(now, before), what
        before = now
    with torch.no_grad():
        for p in params:
            p.data.copy_(p * 1.01)
    moved(".data.copy_")
    params[-1].data = params[-1].data + 0.5
    moved(".data =")
    vector = torch.nn.utils.parameters_to_vector(params).detach() * 0.99
    torch.nn.utils.vector_to_parameters(vector, params)
    moved("vector_to_parameters")
    torch.optim.Adam(params, lr=1e-3, fused=True).step()
    moved("a fused optimizer's step")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        torch._foreach_add_(params, 0.0)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        torch._foreach_add_(params, [p.grad for p in params])
    served("a step captured, not run")
    for _ in range(3):
        g.replay()
        moved("a replayed step")


def test_cuda_brings_the_gradients_along():
    """parameters and gradients that lie elsewhere (here: on the host) come to the model's GPU together, and keep their values"""
    from deepsignal_plant_amd import train_ops as ops
    cfg, m, _ = build(hidden_size=48, num_layers1=1)
    ins, labels = batch(cfg, 20)
    dev = [t.to(DEV) for t in ins]
    m.train()
    ops.cross_entropy(m(*dev)[0], labels.to(DEV)).backward()
    params = m.parameters()
    want = [(p.detach().clone(), p.grad.clone()) for p in params]
    none = params[3]
    none.grad = None
    for p in params:
        grad, p.grad = p.grad, None
        p.data = p.data.cpu()
        p.grad = None if grad is None else grad.cpu()
    m.cuda(0)
    for p, (v, g) in zip(params, want):
        assert torch.equal(p.detach(), v) and (p is none) == (p.grad is None) and (p.grad is None or torch.equal(p.grad, g))
    torch.optim.SGD(params, lr=0.1).step()
    assert torch.equal(m.eval()(*dev)[0], m(*dev)[0])


def test_zero_grad_in_place_and_a_captured_step_that_accumulates():
    """set_to_none=False clears the tensors that are there: a captured backward pass goes on adding to them"""
    from deepsignal_plant_amd import train_ops as ops
    cfg, m, _ = build(hidden_size=48, num_layers1=1)
    ins, labels = batch(cfg, 64)
    dev, y = [t.to(DEV) for t in ins], labels.to(DEV)
    params = m.train().parameters()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torch.autograd.grad(ops.cross_entropy(m(*dev)[0], y), params)
    torch.cuda.current_stream().wait_stream(side)
    for p in params:
        p.grad = torch.zeros_like(p)
    grads = [p.grad for p in params]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for p, d in zip(params, torch.autograd.grad(ops.cross_entropy(m(*dev)[0], y), params)):
            p.grad.add_(d)
    for _ in range(3):
        m.zero_grad(set_to_none=False)
        assert all(p.grad is a and not a.any() for p, a in zip(params, grads))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.grad, w) for p, w in zip(params, want))
    m.zero_grad()
    assert all(p.grad is None for p in params)


def test_a_captured_inference_pass_outlives_the_weights_it_was_captured_with():
    """the parameters move on after the capture: eager calls serve them, the replayed pass still has its own weights and workspace, with
    memory taken and given back in between"""
    cfg, m, _ = build(hidden_size=48, num_layers1=1)
    n = 200
    ins, _ = batch(cfg, n)
    dev = [t.to(DEV) for t in ins]
    m.cuda(0).train().eval()
    m.reserve(n)
    want = [m(*dev)[0].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(*dev)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m(*dev)[0]
        graphs.append((g, out))
        with torch.no_grad():
            for p in m.parameters():
                p.mul_(1.05)
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                m(*dev)
        m.reserve(n)
        want.append(m(*dev)[0].clone())
        assert not torch.equal(want[-1], want[-2])
        m.state_dict()
        assert torch.equal(m(*dev)[0], want[-1])
    for _ in range(3):
        junk = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(8)]
        for (g, out), w in zip(graphs, want):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
        del junk
        torch.cuda.empty_cache()


def test_a_step_captured_into_a_graph():
    """forward, loss, gradients and clipping of one step as a HIP graph: every replay gives the eager result for the inputs that are in the
    buffers by then, with eager work between the replays; two graphs do not share workspaces"""
    from deepsignal_plant_amd import train_ops as ops
    cfg, m, w = build(hidden_size=136, num_layers1=1)
    m.train()
    n = 200
    weight = torch.tensor([1.0, 1.5], device=DEV)
    bufs = [t.to(DEV) for t in batch(cfg, n)[0]]
    y = torch.zeros(n, dtype=torch.int64, device=DEV)
    params = m.parameters()

    def step():
        loss = ops.cross_entropy(m(*bufs)[0], y, weight=weight)
        return (loss.detach(), *ops.clip_grad_norm(torch.autograd.grad(loss, params), 0.1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(4):
        ins, labels = batch(cfg, n, seed=20 + k)
        for b, t in zip(bufs, ins):
            b.copy_(t)
        y.copy_(labels)
        want = step()   # eager, between the replays
        for g, out in (graphs if k % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            for a, b in zip(out[2], want[2]):
                assert torch.equal(a, b)


def test_operators_on_another_stream_and_two_at_once():
    """calls on two streams at once: each its own workspaces, the results those of calls alone"""
    from deepsignal_plant_amd import train_ops as ops
    gen = torch.Generator().manual_seed(1)
    cases = []
    for k in range(2):
        x = torch.randn(60, 9, 40, generator=gen).to(DEV).requires_grad_()
        ws = [((torch.rand(*s, generator=gen) - 0.5) * 0.2).to(DEV).requires_grad_() for _ in range(2) for s in ((600, 40), (600, 150), (600,), (600,))]
        t = torch.randint(0, 5000, (4000,), generator=gen).to(DEV)
        emb = torch.randn(5000, 40, generator=gen).to(DEV).requires_grad_()
        lg, yy = torch.randn(900, 700, generator=gen).to(DEV).requires_grad_(), torch.randint(0, 700, (900,), generator=gen).to(DEV)
        cases.append((x, ws, t, emb, lg, yy))

    def run(c):
        x, ws, t, emb, lg, yy = c
        out = list(torch.autograd.grad(ops.lstm(x, ws)[0].sum(), [x] + ws))
        out += torch.autograd.grad(ops.embedding(t, emb).square().sum(), emb)
        out += torch.autograd.grad(ops.cross_entropy(lg, yy), lg)
        return out + ops.clip_grad_norm(out, 1.0)[1]
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for s, c in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(c))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_second_derivatives_are_refused_not_wrong():
    from deepsignal_plant_amd import train_ops as ops
    w = torch.randn(16, 4, device=DEV, requires_grad=True)
    t = torch.randint(0, 16, (50,), device=DEV)
    g, = torch.autograd.grad(ops.embedding(t, w).square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    x = torch.randn(8, 3, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(ops.cross_entropy(x, torch.zeros(8, dtype=torch.int64, device=DEV)).square(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_what_a_graph_saved_may_not_change():
    """a tensor that a backward pass still needs, changed in place: refused by torch's version count, clipping's writes included"""
    from deepsignal_plant_amd import train_ops as ops
    x = torch.randn(8, 3, device=DEV)
    leaf = x.requires_grad_()
    mid = leaf * 1.0
    loss = ops.cross_entropy(mid, torch.zeros(8, dtype=torch.int64, device=DEV))
    with torch.no_grad():
        mid.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    a = torch.randn(5, device=DEV, requires_grad=True)
    buf = torch.randn(5, device=DEV)
    y = a * buf
    ops.clip_grad_norm([torch.ones(5, device=DEV)], 1.0, out=[buf])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_that_stand_for_their_negative():
    """complex arithmetic behind an operator's output: the gradient that comes back can be a view with its sign still to be turned, also
    one of a single value, which is contiguous"""
    from deepsignal_plant_amd import train_ops as ops
    gen = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    x, y, table, tokens = r(6, 3), torch.tensor([0, 2, 1, 1, 0, 2], device=DEV), r(16, 1), torch.tensor([5], device=DEV)
    w, lw = r(1, 3), [r(4, 3), r(4, 1), r(4), r(4)]
    one = lambda t: (torch.complex(torch.full_like(t, 0.3), t).conj() * (1.5 + 0.5j)).real.sum() * 2.0 + (torch.complex(t, t).conj() * 1j).real.sum()

    def grads(f, leaf, c=None):
        leaf = leaf.clone().requires_grad_()
        return torch.autograd.grad(f(leaf) if c is None else one(f(leaf)), leaf)[0]
    for f, leaf in ((lambda t: ops.cross_entropy(t, y), x), (lambda t: ops.embedding(tokens, t), table), (lambda t: ops.linear(x[:1], t), w),
                    (lambda t: ops.lstm(x[None, :1], [t, *lw[1:]])[0], lw[0])):
        d = torch.tensor(0.0, device=DEV, requires_grad=True)
        k, = torch.autograd.grad(one(d), d)      # `one` is linear: its slope
        assert (grads(f, leaf, 1) - float(k) * grads(lambda t: f(t).sum(), leaf)).abs().max() < 1e-5
    g = torch.complex(r(1), r(1)).conj().imag
    assert g.is_neg() and g.is_contiguous()
    leaf = x.clone().requires_grad_()
    loss = ops.cross_entropy(leaf, y)
    a, b = (torch.autograd.grad(loss, leaf, up.view(()), retain_graph=True)[0] for up in (g, g.resolve_neg()))
    assert torch.equal(a, b)
    assert torch.equal(ops.clip_grad_norm([g], 1e9)[1][0], g.resolve_neg())
    p = torch.nn.Parameter(torch.zeros(1, device=DEV))
    p.grad = torch.complex(r(1), torch.full((1,), 4.0, device=DEV)).conj().imag
    ops.clip_grad_norm_(p, 1.0)
    assert abs(float(p.grad) + 1.0) < 1e-6
