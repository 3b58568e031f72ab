"""The operators of a training step of ModelBiLSTM (deepsignal_plant_amd/train_ops.py) as measured cases: embedding lookup with
its gradient, the LSTM layer with its gradient, weighted cross entropy with its gradient, and clipping by the global gradient
norm.  `run` computes a case in elementary torch operations (own = False) or by the calls a user makes (own = True);
`exact` is the same result in 64 bits, from the definitions."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8, "i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "u8": 1, "i32": 4, "i64": 8}
IGNORE = -100


def listed():
    return [
        # the 13-mers of one training batch of 512 sites through the model's own 16 x 4 table: latency counts
        dict(name="embed_13mers_512", op="embedding", rows=512, cols=13, vocab=16, dim=4, type="f32", tokens="u8", scale=1.0),
        # the same table under the largest batch the forward is run with, 65,536 sites: 852 k tokens fall on 16 rows
        dict(name="embed_13mers_65536", op="embedding", rows=65536, cols=13, vocab=16, dim=4, type="f32", tokens="u8", scale=1.0),
        # a word table: 32 sequences of 4,096 tokens, frequent and rare words, rows scaled by sqrt(dim)
        dict(name="embed_words_bf16", op="embedding", rows=32, cols=4096, vocab=65536, dim=1024, type="bf16", tokens="i64", scale=32.0),
        # one new element of 16 running sequences, the states carried from call to call
        dict(name="lstm_one_token", op="lstm", way="forward", batch=16, steps=1, input=256, hidden=256),
        # a layer of the model's combined stack, one training batch
        dict(name="lstm_comb_512", op="lstm", way="step", batch=512, steps=13, input=512, hidden=256),
        # few long sequences: the recurrence is all there is
        dict(name="lstm_long_32x256", op="lstm", way="step", batch=32, steps=256, input=64, hidden=128),
        # the combined layer under a batch of 4,096 sites
        dict(name="lstm_comb_4096", op="lstm", way="step", batch=4096, steps=13, input=512, hidden=256),
        # the model's two classes, one training batch, the second class weighted
        dict(name="loss_512x2", op="loss", way="step", rows=512, classes=2, type="f32", weighted=True, ignored=0.0),
        # a word model's loss over 8,192 tokens, a tenth of them padding
        dict(name="loss_words_bf16", op="loss", way="step", rows=8192, classes=32000, type="bf16", weighted=False, ignored=0.1),
        # odd sizes: no row but the first is aligned
        dict(name="loss_odd_f32", op="loss", way="step", rows=2049, classes=32001, type="f32", weighted=True, ignored=0.02),
        # the 49 gradients of the default model (4.7 M values)
        dict(name="clip_model_49", op="clip", tensors=49, total=0, type="f32", out="f32", cut=0.1),
        # 290 gradients of very different sizes in bf16, clipped into the 32-bit gradients an optimizer takes
        dict(name="clip_290_bf16", op="clip", tensors=290, total=268435456, type="bf16", out="f32", cut=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("embedding", "lstm", "loss", "clip"))
    if op == "embedding":
        dim = _log(rng, 1, 2048)
        n = _log(rng, 1, min(1 << 20, (131072 * 1024) // dim))
        cols = rng.choice((1, 13, rng.randint(2, 64)))
        vocab = _log(rng, 2, min(200000, (131072 * 1024) // dim))
        return dict(op=op, rows=max(1, n // cols), cols=cols, vocab=vocab, dim=dim, type=rng.choice(("f32", "bf16", "f16")),
                    tokens="u8" if vocab <= 256 and rng.random() < 0.5 else rng.choice(("i32", "i64")), scale=rng.choice((1.0, round(rng.uniform(0.1, 40), 3))))
    if op == "lstm":
        hidden, inputs = _log(rng, 8, 512), _log(rng, 1, 640)
        steps = rng.choice((1, 13, _log(rng, 1, 128)))
        most = 4096 * 13 * 256 * 768 // (steps * hidden * (hidden + inputs))
        return dict(op=op, way=rng.choice(("step", "step", "forward")), batch=_log(rng, 1, max(1, min(8192, most))), steps=steps, input=inputs, hidden=hidden)
    if op == "loss":
        classes = rng.choice((2, _log(rng, 2, 131072), _log(rng, 256, 131072)))
        return dict(op=op, way=rng.choice(("step", "step", "forward")), rows=_log(rng, 1, min(131072, 8192 * 32000 // classes)), classes=classes,
                    type=rng.choice(("f32", "bf16", "f16")), weighted=rng.random() < 0.5, ignored=rng.choice((0.0, 0.1)))
    kind = rng.choice(("f32", "bf16", "f16"))
    tensors = _log(rng, 1, 600)
    return dict(op=op, tensors=tensors, total=max(4 * tensors, _log(rng, 1000, 1 << 28)), type=kind, out=rng.choice((kind, "f32")), cut=rng.choice((0.02, 0.5, 2.0)))


def _sizes(case):
    """numbers of values of the gradients of a clip case: the default model's 49, or sizes over four orders of magnitude"""
    if not case["total"]:
        got = [16 * 4]
        for isz, hid, layers in ((7, 128, 1), (16, 128, 1), (256, 256, 1), (512, 256, 2)):
            got += [4 * hid * isz, 4 * hid * hid, 4 * hid, 4 * hid] * 2 * layers
        return got + [128 * 256, 128, 128 * 256, 128, 256 * 512, 256, 2 * 256, 2]
    n = case["tensors"]
    share = [10.0 ** (-4.0 * ((37 * i) % n) / n) for i in range(n)]
    return [max(1, int(case["total"] * s / sum(share))) for s in share]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = dict(case)
    randn = lambda *shape, type="f32": torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(TYPES[type])
    rand = lambda *shape: torch.rand(*shape, generator=g, device=dev, dtype=torch.float32)
    if case["op"] == "embedding":
        n, v = (case["rows"], case["cols"]), case["vocab"]
        # small tables (bases): every row as often; word tables: the r-th word about as often as 1 / r
        t = (rand(*n) * v).long() if v <= 256 else torch.exp(rand(*n) * math.log(v)).long() - 1
        s["tokens_"] = t.clamp(0, v - 1).to(TYPES[case["tokens"]])
        s["weight_"] = randn(v, case["dim"], type=case["type"]).requires_grad_()
        s["grad_"] = randn(*n, case["dim"], type=case["type"])
    elif case["op"] == "lstm":
        b, t, i, h = case["batch"], case["steps"], case["input"], case["hidden"]
        k = 1.0 / math.sqrt(h)
        leaf = (lambda x: x.requires_grad_()) if case["way"] == "step" else (lambda x: x)
        s["x_"] = leaf(randn(b, t, i))
        s["weights_"] = [leaf((rand(*shape) * 2 - 1) * k) for _ in range(2) for shape in ((4 * h, i), (4 * h, h), (4 * h,), (4 * h,))]
        s["h0_"], s["c0_"] = leaf(randn(2, b, h)), leaf(randn(2, b, h))
        if case["way"] == "step":
            s["grads_"] = [randn(b, t, 2 * h), randn(2, b, h), randn(2, b, h)]
    elif case["op"] == "loss":
        n, c = case["rows"], case["classes"]
        s["logits_"] = (randn(n, c) * 2).to(TYPES[case["type"]])
        if case["way"] == "step":
            s["logits_"].requires_grad_()
        y = (rand(n) * c).long().clamp(0, c - 1)
        y[rand(n) < case["ignored"]] = IGNORE
        y[0] = 0
        s["labels_"] = y
        s["weight_"] = 0.5 + rand(c) if case["weighted"] else None
    else:
        sizes = _sizes(case)
        flat = randn(sum(sizes), type=case["type"])
        s["grads_"] = list(flat.split(sizes))
        s["flat_"] = torch.empty(sum(sizes), device=dev, dtype=TYPES[case["out"]])
        s["out_"] = list(s["flat_"].split(sizes))
        s["max_norm_"] = case["cut"] * math.sqrt(sum(sizes))  # the norm of these gradients is close to sqrt(n)
    return s


def _embedding(s):
    w, g, t = s["weight_"].detach(), s["grad_"], s["tokens_"].long()
    out = (w.float()[t] * s["scale"]).to(w.dtype)
    t, g = t.reshape(-1), g.reshape(-1, w.shape[1])
    # a row named by thousands of tokens: as many short sums of about 64 in 32 bits, joined in 64, lose nothing and do not
    # wait for each other at one place
    parts = t.numel() // (64 * s["vocab"]) if t.numel() > 1024 * s["vocab"] else 1
    if parts > 1:
        t = torch.arange(t.numel(), device=t.device) % parts * s["vocab"] + t
    dw = torch.zeros(parts * s["vocab"], w.shape[1], device=w.device).index_add_(0, t, g.float() * s["scale"])
    return out, (dw.view(parts, *w.shape).sum(0, dtype=torch.float64) if parts > 1 else dw).to(w.dtype)


def _lstm(x, weights, h0, c0):
    """gates of one step = x W_ih^T + b_ih + h W_hh^T + b_hh; the x part of all steps is one product"""
    ends, outs = [], []
    for d in range(2):
        w_ih, w_hh, b_ih, b_hh = weights[4 * d:4 * d + 4]
        xw = x @ w_ih.t() + (b_ih + b_hh)
        h, c, ys = h0[d], c0[d], [None] * x.shape[1]
        for t in (range(x.shape[1]) if d == 0 else reversed(range(x.shape[1]))):
            i, f, g, o = (xw[:, t] + h @ w_hh.t()).chunk(4, 1)
            c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(g)
            h = torch.sigmoid(o) * torch.tanh(c)
            ys[t] = h
        outs.append(torch.stack(ys, 1))
        ends.append((h, c))
    return torch.cat(outs, 2), torch.stack([e[0] for e in ends]), torch.stack([e[1] for e in ends])


def _loss(s):
    logits, y = s["logits_"].detach(), s["labels_"]
    x = logits.float()
    live = y != IGNORE
    at = torch.where(live, y, 0)[:, None]
    w = live.float() if s["weight_"] is None else torch.where(live, s["weight_"][at[:, 0]], 0.0)
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    total = w.double().sum()
    loss = ((torch.log(z) + m - x.gather(1, at))[:, 0].double() * w).sum() / total
    if s["way"] == "forward":
        return (loss.float(),)
    k = (w / total.float())[:, None]
    return loss.float(), (e * (k / z)).scatter_add_(1, at, -k).to(logits.dtype)


def _clip(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads_"]]).sum().sqrt()
    k = (s["max_norm_"] / (norm + 1e-6)).clamp(max=1.0).float()
    torch._foreach_copy_(s["out_"], [g.float() * k for g in s["grads_"]])
    return norm.float()


def run(s):
    if own:
        from deepsignal_plant_amd import train_ops as ops
    if s["op"] == "embedding":
        if not own:
            out, dw = _embedding(s)
        else:
            out = ops.embedding(s["tokens_"], s["weight_"], scale=s["scale"])
            dw, = torch.autograd.grad(out, s["weight_"], s["grad_"])
        return {"out": out, "weight_grad": dw}
    if s["op"] == "lstm":
        layer = ops.lstm if own else _lstm
        if s["way"] == "forward":
            with torch.no_grad():
                return dict(zip(("y", "hn", "cn"), layer(s["x_"], s["weights_"], s["h0_"], s["c0_"])))
        outs = layer(s["x_"], s["weights_"], s["h0_"], s["c0_"])
        grads = torch.autograd.grad(outs, [s["x_"], s["h0_"], s["c0_"]] + s["weights_"], s["grads_"])
        return {"outs": list(outs), "grads": list(grads)}
    if s["op"] == "loss":
        if not own:
            return dict(zip(("loss", "grad"), _loss(s)))
        loss = ops.cross_entropy(s["logits_"], s["labels_"], weight=s["weight_"], ignore_index=IGNORE)
        if s["way"] == "forward":
            return {"loss": loss}
        return {"loss": loss, "grad": torch.autograd.grad(loss, s["logits_"])[0]}
    norm = ops.clip_grad_norm(s["grads_"], s["max_norm_"], out=s["out_"])[0] if own else _clip(s)
    return {"norm": norm, "grads": s["flat_"]}


def work(case):
    if case["op"] == "embedding":
        # forward: tokens and the rows they name in (no more than the table has), the output out; backward: gradient and tokens in, the table's gradient out
        n, sz = case["rows"] * case["cols"], SIZE[case["type"]]
        rows = min(n, case["vocab"])
        return {"bytes": n * (2 * case["dim"] * sz + SIZE[case["tokens"]]) + (rows + case["vocab"]) * case["dim"] * sz, "flops": 2 * n * case["dim"]}
    if case["op"] == "lstm":
        b, t, i, h = case["batch"], case["steps"], case["input"], case["hidden"]
        states, params = 2 * 2 * b * h, 2 * 4 * h * (i + h + 2)
        product = 2 * 2 * b * t * 4 * h * (i + h)
        one = b * t * (i + 2 * h) + 2 * states + params
        # backward: the same products for the inputs' gradients and once more for the weights'; y's gradient in, x's, the states' and the weights' out
        return {"bytes": 4 * one * (1 if case["way"] == "forward" else 2), "flops": product * (1 if case["way"] == "forward" else 3)}
    if case["op"] == "loss":
        n, c, sz = case["rows"], case["classes"], SIZE[case["type"]]
        passes = 1 if case["way"] == "forward" else 2
        return {"bytes": n * c * sz * passes + 8 * n + (4 * c if case["weighted"] else 0), "flops": 4 * n * c * passes}
    n = sum(_sizes(case))
    return {"bytes": n * (SIZE[case["type"]] + SIZE[case["out"]]), "flops": 3 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        t, w = s["tokens_"].reshape(-1).long(), s["weight_"].detach()
        out = torch.index_select(w, 0, t).double().mul_(case["scale"]).view(*s["tokens_"].shape, -1)
        order = torch.argsort(t, stable=True)
        edges = torch.searchsorted(t[order], torch.arange(case["vocab"] + 1, device=t.device))
        dw = torch.empty(w.shape, dtype=torch.float64, device=w.device)
        step = max(1, (1 << 26) // max(1, t.numel()))  # columns at a time: sums of a row's tokens as differences would lose digits, segments do not
        for at in range(0, w.shape[1], step):
            part = s["grad_"].reshape(t.numel(), -1)[:, at:at + step][order].double()
            dw[:, at:at + step] = torch.segment_reduce(part, "sum", offsets=edges, axis=0, initial=0.0)
        return {"out": out, "weight_grad": dw * case["scale"]}
    if case["op"] == "lstm":
        return _exact_lstm(case, s)
    if case["op"] == "loss":
        logits, y = s["logits_"].detach(), s["labels_"]
        live = torch.nonzero(y != IGNORE)[:, 0]
        w = torch.ones(case["classes"], device=y.device) if s["weight_"] is None else s["weight_"]
        w = w.double()[y[live]]
        grad = torch.zeros(logits.shape, dtype=torch.float64, device=y.device) if case["way"] == "step" else None
        loss, step = torch.zeros((), dtype=torch.float64, device=y.device), max(1, (1 << 25) // case["classes"])
        for at in range(0, len(live), step):
            r, k = live[at:at + step], w[at:at + step]
            lp = torch.log_softmax(logits[r].double(), 1)
            own_class = y[r][:, None]
            loss -= (lp.gather(1, own_class)[:, 0] * k).sum()
            if grad is not None:
                p = lp.exp_()
                p.scatter_add_(1, own_class, torch.full_like(p[:, :1], -1.0))
                grad[r] = p * (k / w.sum())[:, None]
        return {"loss": loss / w.sum(), **({"grad": grad} if grad is not None else {})}
    flat = torch.cat(s["grads_"]).double()
    norm = flat.norm()
    return {"norm": norm, "grads": flat * min(1.0, s["max_norm_"] / (float(norm) + 1e-6))}


def _exact_lstm(case, s):
    """forward and backpropagation through time written out, in 64 bits"""
    x = s["x_"].detach().double()
    b, t, i, h = case["batch"], case["steps"], case["input"], case["hidden"]
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=x.device)
    y, hn, cn, dx, dh0, dc0, dws = new(b, t, 2 * h), new(2, b, h), new(2, b, h), new(b, t, i), new(2, b, h), new(2, b, h), []
    for d in range(2):
        w_ih, w_hh, b_ih, b_hh = (p.detach().double() for p in s["weights_"][4 * d:4 * d + 4])
        order = list(range(t))[::-1 if d else 1]
        hs, cs, acts = s["h0_"][d].detach().double(), s["c0_"][d].detach().double(), []
        for k in order:
            z = torch.addmm(b_ih + b_hh, x[:, k], w_ih.T).addmm_(hs, w_hh.T)
            a = z.sigmoid()
            a[:, 2 * h:3 * h] = z[:, 2 * h:3 * h].tanh()
            new_c = a[:, h:2 * h] * cs + a[:, :h] * a[:, 2 * h:3 * h]
            acts.append((k, a, hs, cs, new_c))
            hs, cs = a[:, 3 * h:] * new_c.tanh(), new_c
            y[:, k, d * h:(d + 1) * h] = hs
        hn[d], cn[d] = hs, cs
        if case["way"] == "forward":
            continue
        gy, ghn, gcn = (g.double() for g in s["grads_"])
        dh, dc, dwi, dwh, db = ghn[d], gcn[d], new(4 * h, i), new(4 * h, h), new(4 * h)
        for k, a, hp, cp, c in reversed(acts):
            dh = dh + gy[:, k, d * h:(d + 1) * h]
            ai, af, ag, ao, tc = a[:, :h], a[:, h:2 * h], a[:, 2 * h:3 * h], a[:, 3 * h:], c.tanh()
            dc = dc + dh * ao * (1 - tc * tc)
            dz = torch.cat((dc * ag * ai * (1 - ai), dc * cp * af * (1 - af), dc * ai * (1 - ag * ag), dh * tc * ao * (1 - ao)), 1)
            dwi += dz.T @ x[:, k]
            dwh += dz.T @ hp
            db += dz.sum(0)
            dx[:, k] += dz @ w_ih
            dh, dc = dz @ w_hh, dc * af
        dh0[d], dc0[d] = dh, dc
        dws += [dwi, dwh, db, db.clone()]
    if case["way"] == "forward":
        return {"y": y, "hn": hn, "cn": cn}
    return {"outs": [y, hn, cn], "grads": [dx, dh0, dc0] + dws}
