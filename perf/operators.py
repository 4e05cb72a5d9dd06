"""Measured cases of the operators on learned node representations: embedding lookup with its
gradient, dropout from the counter-based streams, and softmax cross entropy over the node
vocabulary.  ``run`` computes them either through this package (``own`` true) or in a plain form
of elementary tensor operations."""
import math

import torch

own = False

# the graph sizes this repository is benchmarked on
PRODUCTS = 2449029
REDDIT = 232965

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # serving: the vector of one node out of a table of a whole graph
        dict(name="embed_one", op="embedding", grad="none", n=1, V=PRODUCTS, D=100, dtype="fp32", scale=1.0, skew=1.0),
        # the frontier of a sampled super-batch over learned features, trained with a dense gradient
        dict(name="embed_frontier", op="embedding", grad="dense", n=1000003, V=REDDIT, D=100, dtype="fp32",
             scale=1.0, skew=2.0),
        # every position of a walk corpus (hubs repeat by the thousand), scaled by sqrt(D)
        dict(name="embed_walks", op="embedding", grad="dense", n=4000000, V=PRODUCTS, D=128, dtype="bf16",
             scale=11.313708498984761, skew=4.0),
        # one minibatch against a large table: only the touched rows have a gradient
        dict(name="embed_sparse", op="embedding", grad="sparse", n=65537, V=PRODUCTS, D=64, dtype="fp16",
             scale=1.0, skew=2.0),
        # the input rows of a small minibatch
        dict(name="drop_small", op="dropout", grad="none", rows=512, D=100, dtype="fp32", p=0.5),
        # hidden rows of a super-batch, odd width, both directions
        dict(name="drop_hidden", op="dropout", grad="dense", rows=300007, D=99, dtype="fp16", p=0.1),
        # the gathered rows of a large frontier, both directions
        dict(name="drop_frontier", op="dropout", grad="dense", rows=4000000, D=100, dtype="bf16", p=0.3),
        # serving: the log-probability of one node against the whole vocabulary
        dict(name="loss_one", op="loss", grad="none", n=1, V=PRODUCTS, D=128, dtype="bf16", scale=1.0, ignored=0.0),
        # node classification over a super-batch: many rows, few classes
        dict(name="loss_classes", op="loss", grad="dense", n=300007, V=47, D=256, dtype="bf16", scale=1.0, ignored=0.5),
        # 32-bit embeddings of a small graph
        dict(name="loss_fp32", op="loss", grad="dense", n=4000, V=50021, D=64, dtype="fp32", scale=1.0, ignored=0.1),
        # one minibatch of 1024 seeds against a middle-sized vocabulary, odd width, a temperature
        dict(name="loss_minibatch", op="loss", grad="dense", n=1024, V=REDDIT, D=100, dtype="fp16", scale=0.5,
             ignored=0.05),
        # walk corpus: full softmax over all nodes of the large graph
        dict(name="loss_walks", op="loss", grad="dense", n=8192, V=PRODUCTS, D=128, dtype="bf16", scale=1.0,
             ignored=0.02),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "dropout", "loss", "loss"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "embedding":
        grad = rng.choice(["none", "dense", "sparse"])
        return dict(op=op, grad=grad, n=_log_int(rng, 1, 2000000), V=_log_int(rng, 100, PRODUCTS),
                    D=_log_int(rng, 16, 256), dtype=dtype, scale=rng.choice([1.0, 0.25, 8.0]),
                    skew=rng.choice([1.0, 2.0, 4.0]))
    if op == "dropout":
        return dict(op=op, grad=rng.choice(["none", "dense"]), rows=_log_int(rng, 1, 1500000), D=_log_int(rng, 1, 256),
                    dtype=dtype, p=rng.choice([0.1, 0.25, 0.5, 0.9]))
    while True:
        n, V, D = _log_int(rng, 1, 300000), _log_int(rng, 2, PRODUCTS), _log_int(rng, 16, 256)
        # no more work than the largest listed case; 32-bit products cost what 16-bit ones do not
        if n * V * D <= (8192 * PRODUCTS * 128 // (8 if dtype == "fp32" else 1)):
            break
    return dict(op=op, grad=rng.choice(["none", "dense", "dense"]), n=n, V=V, D=D, dtype=dtype,
                scale=rng.choice([1.0, 1.0, 0.5]), ignored=rng.choice([0.0, 0.05, 0.5]))


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(rows, cols, std):
        t = torch.empty((rows, cols), dtype=dt, device=dev)
        return t.normal_(0.0, std, generator=gen)

    state = dict(case=dict(case), dtype=dt)
    needs = case["grad"] != "none"
    if case["op"] == "embedding":
        n, V, D = case["n"], case["V"], case["D"]
        state["weight"] = normal(V, D, D ** -0.5).requires_grad_(needs)
        # a few nodes are looked up far more often than the rest, as node degrees are skewed; about 1
        # in 50 positions is "no node".  How often the nodes occur is the case's; which nodes they
        # are and where they stand is the seed's, so that the number of distinct ones is the case's.
        often = torch.Generator(device=dev)
        often.manual_seed(5)
        u = torch.rand(n, generator=often, device=dev, dtype=torch.float64)
        idx = (u.pow(case["skew"]) * V).long().clamp_(0, V - 1)
        first = int(torch.randint(0, V, (1,), generator=gen, device=dev))
        idx = (idx + first) % V
        if n > 1:
            idx[torch.rand(n, generator=often, device=dev) < 0.02] = -1
        state["index"] = idx[torch.randperm(n, generator=gen, device=dev)]
        if needs:
            state["grad"] = normal(n, D, 1.0)
    elif case["op"] == "dropout":
        state["x"] = normal(case["rows"], case["D"], 1.0).requires_grad_(needs)
        state["seed"] = int(seed) * 7919 + 11
        state["stream"] = int(seed) % 1000
        if needs:
            state["grad"] = normal(case["rows"], case["D"], 1.0)
    else:
        n, V, D = case["n"], case["V"], case["D"]
        # logits with a standard deviation of about 2, as trained representations give
        state["x"] = normal(n, D, 2.0).requires_grad_(needs)
        state["weight"] = normal(V, D, D ** -0.5).requires_grad_(needs)
        t = (torch.rand(n, generator=gen, device=dev, dtype=torch.float64).square() * V).long().clamp_(0, V - 1)
        if case["ignored"] > 0 and n > 1:
            t[torch.rand(n, generator=gen, device=dev) < case["ignored"]] = -1
        state["target"] = t
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import gsampler_b200 as gs

    case = state["case"]
    if case["op"] == "embedding":
        out = gs.ops.embedding(state["weight"], state["index"], scale=case["scale"], padding_idx=-1,
                               sparse=case["grad"] == "sparse")
        if case["grad"] == "none":
            return out
        (dw,) = torch.autograd.grad(out, [state["weight"]], state["grad"])
        if case["grad"] == "sparse":
            return out.detach(), dw.indices()[0], dw.values()
        return out.detach(), dw
    if case["op"] == "dropout":
        out = gs.ops.dropout(state["x"], case["p"], seed=state["seed"], stream=state["stream"])
        if case["grad"] == "none":
            return out
        (dx,) = torch.autograd.grad(out, [state["x"]], state["grad"])
        return out.detach(), dx
    if case["grad"] == "none":
        return gs.ops.linear_cross_entropy(state["x"], state["weight"], state["target"], scale=case["scale"],
                                           reduction="none")
    loss = gs.ops.linear_cross_entropy(state["x"], state["weight"], state["target"], scale=case["scale"])
    dx, dw = torch.autograd.grad(loss, [state["x"], state["weight"]])
    return loss.detach(), dx, dw


# ------------------------------------------------------------------ plain form
def _keep_mask(total, seed, stream, p, dev):
    """Philox4x32-10 by 64-bit integer operations; eight 16-bit numbers a block."""
    m32 = 0xFFFFFFFF
    g = torch.arange((total + 7) // 8, device=dev, dtype=torch.int64)
    c0, c1, c2, c3 = g & m32, g >> 32, torch.zeros_like(g), torch.full_like(g, stream & m32)
    k0, k1 = seed & m32, (seed >> 32) & m32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & m32) ^ c1 ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c3 ^ k1, p0 & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    halves = torch.stack([c0 & 65535, c0 >> 16, c1 & 65535, c1 >> 16, c2 & 65535, c2 >> 16, c3 & 65535, c3 >> 16], 1)
    return halves.flatten()[:total] >= int(round(p * 65536))


def _run_plain(state):
    with torch.no_grad():
        case = state["case"]
        if case["op"] == "embedding":
            return _plain_embedding(state, case)
        if case["op"] == "dropout":
            return _plain_dropout(state, case)
        return _plain_loss(state, case)


def _plain_embedding(state, case):
    w, idx, dt = state["weight"], state["index"], state["dtype"]
    live = idx >= 0
    rows = w[idx.clamp(min=0)].float() * case["scale"]
    out = torch.where(live[:, None], rows, 0.0).to(dt)
    del rows
    if case["grad"] == "none":
        return out
    g = torch.where(live[:, None], state["grad"].float(), 0.0)
    if case["grad"] == "dense":
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        dw.index_add_(0, idx.clamp(min=0), g)
        return out, (dw * case["scale"]).to(dt)
    ids, place = torch.unique(idx[live], return_inverse=True)
    dw = torch.zeros((ids.numel(), w.shape[1]), dtype=torch.float32, device=w.device)
    dw.index_add_(0, place, g[live])
    return out, ids, (dw * case["scale"]).to(dt)


def _plain_dropout(state, case):
    x, dt = state["x"], state["dtype"]
    keep = _keep_mask(x.numel(), state["seed"], state["stream"], case["p"], x.device).view(x.shape)
    mul = 65536.0 / (65536 - int(round(case["p"] * 65536)))
    out = torch.where(keep, x.float() * mul, 0.0).to(dt)
    if case["grad"] == "none":
        return out
    return out, torch.where(keep, state["grad"].float() * mul, 0.0).to(dt)


def _plain_loss(state, case):
    x, w, t, dt, s = state["x"].float(), state["weight"], state["target"], state["dtype"], case["scale"]
    n, V = x.shape[0], w.shape[0]
    live = t >= 0
    piece = max(1, min(V, (1 << 29) // n))
    m = torch.full((n,), -math.inf, device=x.device)
    z = torch.zeros(n, device=x.device)
    for v0 in range(0, V, piece):
        l = (x @ w[v0:v0 + piece].float().t()) * s
        m2 = torch.maximum(m, l.amax(1))
        z = z * torch.exp(m - m2) + torch.exp(l - m2[:, None]).sum(1)
        m = m2
        del l
    lse = m + torch.log(z)
    wt = w[t.clamp(min=0)].float()
    loss = torch.where(live, lse - (x * wt).sum(1) * s, 0.0)
    if case["grad"] == "none":
        return loss
    count = live.sum().clamp(min=1)
    g = live.float() / count
    dx = torch.zeros_like(x)
    dw = torch.empty(w.shape, dtype=dt, device=x.device)
    ids = torch.arange(V, device=x.device)
    for v0 in range(0, V, piece):
        wp = w[v0:v0 + piece].float()
        p = torch.exp((x @ wp.t()) * s - lse[:, None])
        p.sub_((t[:, None] == ids[None, v0:v0 + piece]).float()).mul_(g[:, None] * s)
        dx += p @ wp
        dw[v0:v0 + piece] = (p.t() @ x).to(dt)
        del p
    return loss.sum() / count, dx.to(dt), dw


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        if case["op"] == "embedding":
            W, i = state["weight"], state["index"]
            here = (i != -1).nonzero().squeeze(1)
            out = torch.zeros((i.numel(), case["D"]), dtype=torch.float64, device=W.device)
            out[here] = W[i[here]].double().mul_(case["scale"])
            if case["grad"] == "none":
                return out
            summed = torch.zeros((case["V"], case["D"]), dtype=torch.float64, device=W.device)
            for a in range(0, here.numel(), 1 << 20):
                h = here[a:a + (1 << 20)]
                summed.index_add_(0, i[h], state["grad"][h].double())
            summed.mul_(case["scale"])
            if case["grad"] == "dense":
                return out, summed
            touched = torch.zeros(case["V"], dtype=torch.bool, device=W.device)
            touched[i[here]] = True
            ids = touched.nonzero().squeeze(1)
            return out, ids, summed[ids]
        if case["op"] == "dropout":
            total = case["rows"] * case["D"]
            parts = []
            for a in range(0, total, 1 << 26):  # word by word, each position's own block
                e = torch.arange(a, min(total, a + (1 << 26)), device="cuda")
                parts.append(_word16(e, state["seed"], state["stream"]))
            level = round(case["p"] * 65536)
            kept = (torch.cat(parts) >= level).double().view(case["rows"], case["D"]) / (1.0 - level / 65536.0)
            out = kept * state["x"].double()
            return out if case["grad"] == "none" else (out, kept.mul_(state["grad"].double()))
        return _exact_loss(case, state)


def _word16(e, seed, stream):
    c = [(e // 8) % 2 ** 32, (e // 8) // 2 ** 32, e * 0, e * 0 + stream]
    key = [seed % 2 ** 32, (seed // 2 ** 32) % 2 ** 32]
    for _ in range(10):
        # a 32 x 32 bit product in 16-bit limbs, so that nothing passes 63 bits
        def product(a, k):
            low = a * (k % 65536)
            high = a * (k // 65536)
            whole_low = low + (high % 65536) * 65536
            return (high // 65536) + whole_low // 2 ** 32, whole_low % 2 ** 32

        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    j = e % 8
    word = torch.where(j < 4, torch.where(j < 2, c[0], c[1]), torch.where(j < 6, c[2], c[3]))
    return torch.where(j % 2 == 0, word % 65536, word // 65536)


def _exact_loss(case, state):
    n, V, s = case["n"], case["V"], case["scale"]
    X, W, t = state["x"].double(), state["weight"], state["target"]
    counted = t != -1
    step = max(1, (1 << 28) // n)
    pieces = [(a, min(V, a + step)) for a in range(0, V, step)]
    tops, sums = [], []
    for a, b in pieces:
        logits = torch.mm(X, W[a:b].double().T).mul_(s)
        tops.append(logits.max(dim=1).values)
        sums.append(logits.sub_(tops[-1][:, None]).exp_().sum(1))
    tops, sums = torch.stack(tops), torch.stack(sums)
    top = tops.max(dim=0).values
    lse = top + ((tops - top).exp() * sums).sum(0).log()
    target_rows = W[torch.where(counted, t, 0)].double()
    loss = (lse - s * torch.einsum("nd,nd->n", X, target_rows)) * counted
    if case["grad"] == "none":
        return loss
    number = max(1, int(counted.sum()))
    pull = counted.double() * (s / number)
    dX = -target_rows
    dW = torch.empty((V, case["D"]), dtype=torch.float64, device=X.device)
    pulled = X * pull[:, None]
    for a, b in pieces:
        wp = W[a:b].double()
        prob = torch.mm(X, wp.T).mul_(s).sub_(lse[:, None]).exp_()
        dX += prob @ wp
        dW[a:b] = prob.T @ pulled
    dW.index_add_(0, t[counted], -pulled[counted])
    return loss.sum() / number, dX * pull[:, None], dW


# ------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "embedding":
        n, V, D = case["n"], case["V"], case["D"]
        # rows that are looked up at least once (each is read once)
        distinct = V * sum(1.0 - math.exp(-n / V * d) for d in _densities(case["skew"])) / len(_densities(case["skew"]))
        distinct = max(1.0, min(distinct, float(n)))
        total = 8 * n + (distinct + n) * D * size
        flops = n * D
        if case["grad"] != "none":
            rows = V if case["grad"] == "dense" else distinct
            total += n * D * size + rows * D * size + (8 * rows if case["grad"] == "sparse" else 0)
            flops += n * D
        return {"bytes": int(total), "flops": int(flops)}
    if case["op"] == "dropout":
        total = case["rows"] * case["D"]
        ways = 1 if case["grad"] == "none" else 2
        return {"bytes": 2 * size * total * ways, "flops": total * ways}
    n, V, D = case["n"], case["V"], case["D"]
    moved = (n + V) * D * size + 8 * n
    if case["grad"] == "none":
        return {"bytes": moved + 4 * n, "flops": 2 * n * V * D}
    return {"bytes": moved + (n + V) * D * size, "flops": 6 * n * V * D}


def _densities(skew, points=200):
    """Relative frequency of the ids at the midpoints of [0, 1) under u ** skew."""
    return [(1.0 / skew) * ((k + 0.5) / points) ** (1.0 / skew - 1.0) for k in range(points)]
