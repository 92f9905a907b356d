"""What the token-model operators of vortex_amd are measured on: the two ends of a language model around its network.

    embed        out[t] = scale * table[ids[t]]                              (ids < 0 are padding: a row of zeros)
    embed_grad   d_table[v] = scale * sum of grad_out[t] over ids[t] == v
    linear       y[m,n] = s[m] * sw[n] * sum_k q[m,k] qw[n,k] (+ bias[n]),  q = rint(127 x / max|x|) for each token m
    verify       drafted tokens against the target's softmax, from given uniform numbers

`run` computes an operator in elementary torch operations, or with `own` by the framework's entry points."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the tokens of one decoding step of a few sequences: the smallest call there is, latency alone
        {"name": "embed 4 tokens", "op": "embed", "T": 4, "V": 32000, "D": 1024, "dtype": "bf16", "pad": 0.0, "scale": 32.0},
        # a prefill batch, right-padded
        {"name": "embed prefill", "op": "embed", "T": 32768, "V": 131072, "D": 4096, "dtype": "bf16", "pad": 0.1, "scale": 1.0},
        # one micro-batch of a small model's training step
        {"name": "grad micro-batch f32", "op": "embed_grad", "T": 2048, "V": 32000, "D": 1024, "dtype": "f32", "pad": 0.0, "scale": 32.0},
        # odd vocabulary and width, padded sequences
        {"name": "grad odd f16", "op": "embed_grad", "T": 5001, "V": 50021, "D": 1000, "dtype": "f16", "pad": 0.2, "scale": 1.0},
        # a full training batch over a large vocabulary
        {"name": "grad large bf16", "op": "embed_grad", "T": 65536, "V": 131072, "D": 4096, "dtype": "bf16", "pad": 0.0, "scale": 1.0},
        # the vocabulary head on one token
        {"name": "head 1 token", "op": "linear", "M": 1, "N": 32000, "K": 4096, "dtype": "bf16", "out": "bf16", "bias": False},
        # a verification batch through a head of odd sizes
        {"name": "head 37 tokens odd", "op": "linear", "M": 37, "N": 50021, "K": 1000, "dtype": "f16", "out": "f32", "bias": True},
        # the 1x1 convolution in front of the coarse YOLO layer as a product: 256 images of 13 x 13 cells, 255 channels
        {"name": "yolo head 1x1", "op": "linear", "M": 43264, "N": 255, "K": 1024, "dtype": "f32", "out": "f32", "bias": True},
        # a long prompt through a wide projection: bound by the matrix cores
        {"name": "projection 8192 tokens", "op": "linear", "M": 8192, "N": 16384, "K": 4096, "dtype": "bf16", "out": "bf16", "bias": False},
        # one sequence with four drafts: latency
        {"name": "verify 1 sequence", "op": "verify", "B": 1, "K": 4, "V": 32000, "dtype": "bf16", "draft": True, "greedy": 0.0, "ragged": False},
        # drafts looked up in the prompt (no draft distribution), ragged, a third of the sequences greedy, odd vocabulary
        {"name": "verify lookup ragged f32", "op": "verify", "B": 33, "K": 7, "V": 50021, "dtype": "f32", "draft": False, "greedy": 0.34, "ragged": True},
        # a serving batch over a large vocabulary
        {"name": "verify 64 sequences", "op": "verify", "B": 64, "K": 5, "V": 131072, "dtype": "bf16", "draft": True, "greedy": 0.0, "ragged": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "linear", "verify"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    case = {"op": op, "dtype": dtype}
    if op == "embed":
        case.update(T=_log(rng, 1, 32768), V=_log(rng, 1000, 131072), D=_log(rng, 64, 4096), pad=rng.choice([0.0, 0.3]), scale=rng.choice([1.0, 32.0, 0.125]))
    elif op == "embed_grad":
        case.update(T=_log(rng, 1, 32768), V=_log(rng, 1000, 131072), D=_log(rng, 64, 2048), pad=rng.choice([0.0, 0.3]), scale=rng.choice([1.0, 32.0, 0.125]))
    elif op == "linear":
        case.update(M=_log(rng, 1, 8192), N=_log(rng, 100, 16384), K=_log(rng, 64, 4096), out=rng.choice(["f32", "bf16", "f16"]), bias=rng.random() < 0.5)
        if rng.random() < 0.7:
            case["K"] = max(64, case["K"] // 64 * 64)
    else:
        case.update(B=_log(rng, 1, 32), K=rng.randint(1, 8), V=_log(rng, 1000, 131072), draft=rng.random() < 0.6, greedy=rng.choice([0.0, 0.3]), ragged=rng.random() < 0.5)
    return case


def _tokens(n, V, gen):
    """Token ids as text has them: the n-th most frequent one about 1/n as often as the first."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dt = DTYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if op in ("embed", "embed_grad"):
        T, V, D = case["T"], case["V"], case["D"]
        ids = _tokens(T, V, gen)
        if case["pad"]:
            ids = torch.where(uniform(T) < case["pad"], torch.full_like(ids, -1), ids)
        s["ids"] = ids
        if op == "embed":
            s["table"] = (normal(V, D) * 0.02).to(dt)
        else:
            s["grad_out"] = (normal(T, D) * 0.01).to(dt)
    elif op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        # activations with a few large channels, weights quantised once for each output channel
        s["x"] = (normal(M, K) * (1.0 + 7.0 * (uniform(K) < 0.01).float())).to(dt)
        w = normal(N, K) * 0.02
        amax = w.abs().amax(1)
        s["qw"] = torch.round(w * (127.0 / amax)[:, None]).clamp_(-127, 127).to(torch.int8)
        s["sw"] = amax / 127.0
        s["bias"] = normal(N) * 0.1 if case["bias"] else None
    else:
        B, K, V = case["B"], case["K"], case["V"]
        target = normal(B, K + 1, V) * 2.5
        draft = target[:, :K] + normal(B, K, V) * 0.7              # a drafter that is nearly right
        noise = -torch.log(-torch.log(uniform(B, K, V).clamp_(1e-20, 1.0 - 1e-7)))
        s["temperature"] = torch.where(uniform(B) < case["greedy"], torch.zeros(B, device="cuda"), 0.5 + uniform(B))
        t = s["temperature"].clamp_min(1e-3)[:, None, None]
        draft = draft.to(dt)
        s["draft_tokens"] = (draft.float() / t + noise * (s["temperature"] > 0)[:, None, None]).argmax(-1)
        s["target"] = target.to(dt)
        s["draft"] = draft if case["draft"] else None
        s["uniforms"] = uniform(B, K + 1)
        s["lens"] = torch.randint(0, K + 1, (B,), generator=gen, device="cuda", dtype=torch.int32) if case["ragged"] else None
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _embed(s):
    ids, table = s["ids"], s["table"]
    rows = table[ids.clamp_min(0)].float() * s["case"]["scale"]
    return torch.where((ids >= 0)[:, None], rows, torch.zeros((), device=rows.device)).to(table.dtype)


def _embed_grad(s):
    ids, g, V = s["ids"], s["grad_out"], s["case"]["V"]
    out = torch.zeros(V + 1, g.size(1), device=g.device)           # the last row takes the padding
    out.index_add_(0, torch.where(ids < 0, torch.full_like(ids, V), ids), g.float())
    return (out[:V] * s["case"]["scale"]).to(g.dtype)


def _linear(s):
    x = s["x"].double()                                            # a quotient next to a half decides an integer
    amax = x.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, torch.round(x * 127.0 / amax), torch.zeros_like(x)).float()
    y = (q @ s["qw"].float().t()) * ((amax.float() / 127.0) * s["sw"][None])
    if s["bias"] is not None:
        y = y + s["bias"][None]
    return y.to(DTYPES[s["case"]["out"]])


def _softmax64(x, t):
    z = (x - x.amax(-1, keepdim=True)) / t
    e = torch.exp(z)
    return e / e.sum(-1, keepdim=True)


def _verify(s):
    # 64 bits: a token is a whole number, decided by where a cumulative sum passes a border
    target, draft, x, u = s["target"].double(), s["draft"], s["draft_tokens"], s["uniforms"].double()
    B, K = x.shape
    V = target.size(-1)
    dev = target.device
    lens = s["lens"].long() if s["lens"] is not None else torch.full((B,), K, device=dev)
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None, None]
    p = _softmax64(target, t)
    best = target.argmax(-1)
    onehot = torch.zeros(B, K, V, device=dev, dtype=torch.float64).scatter_(2, x[..., None], 1.0) if draft is None else None
    q = onehot if draft is None else _softmax64(draft.double(), t)
    px, qx = p[:, :K].gather(2, x[..., None])[..., 0], q.gather(2, x[..., None])[..., 0]
    same = best[:, :K] == x
    ok = torch.where(greedy[:, None], same, u[:, :K] * qx < px)
    ratio = torch.where(greedy[:, None], same.double(), torch.clamp(px / qx, max=1.0))
    used = torch.arange(K, device=dev)[None] < lens[:, None]
    n = (ok & used).long().cumprod(1).sum(1)                       # accepted drafts
    rows = torch.arange(B, device=dev)
    r = p[rows, n]
    r = torch.where((n < lens)[:, None], (r - q[rows, n.clamp_max(K - 1)]).clamp_min(0.0), r)
    c = r.cumsum(1)
    nxt = (c <= u[:, K:] * c[:, -1:]).sum(1).clamp_max(V - 1)
    nxt = torch.where(greedy, best[rows, n], nxt)
    at = torch.arange(K + 1, device=dev)[None]
    tokens = torch.where(at < n[:, None], torch.cat((x, x[:, :1]), 1), torch.full((B, K + 1), -1, device=dev))
    tokens = torch.where(at == n[:, None], nxt[:, None], tokens)
    return {"tokens": tokens, "counts": (n + 1).int(), "accept": torch.where(used, ratio, torch.zeros_like(ratio)).float()}


def run(state):
    op = state["case"]["op"]
    if own:
        from vortex_amd import ops
        if op == "embed":
            return ops.embed_tokens(state["ids"], state["table"], state["case"]["scale"])
        if op == "embed_grad":
            return ops.embed_tokens_grad(state["ids"], state["grad_out"], state["case"]["V"], state["case"]["scale"])
        if op == "linear":
            return ops.linear_w8a8(state["x"], state["qw"], state["sw"], state["bias"], DTYPES[state["case"]["out"]])
        tokens, counts, accept, _ = ops.verify_drafts(state["target"], state["draft_tokens"], state["uniforms"],
                                                      draft_logits=state["draft"], draft_lens=state["lens"], temperature=state["temperature"])
        return {"tokens": tokens, "counts": counts, "accept": accept}
    return {"embed": _embed, "embed_grad": _embed_grad, "linear": _linear, "verify": _verify}[op](state)


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "embed":
        n = case["T"] * case["D"]
        return {"bytes": 8 * case["T"] + 2 * n * e, "flops": n}
    if case["op"] == "embed_grad":
        n = case["T"] * case["D"]
        return {"bytes": 8 * case["T"] + n * e + case["V"] * case["D"] * e, "flops": n}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K * e + N * K + 4 * N + M * N * SIZE[case["out"]], "flops": 2 * M * N * K}
    rows = case["B"] * (case["K"] + 1 + (case["K"] if case["draft"] else 0))
    return {"bytes": rows * case["V"] * e, "flops": 4 * rows * case["V"]}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        table = torch.cat((s["table"].double() * case["scale"], torch.zeros(1, case["D"], device="cuda", dtype=torch.float64)))
        return table.index_select(0, s["ids"] % (case["V"] + 1))   # -1 falls on the row of zeros
    if op == "embed_grad":
        # running sums over the tokens in the order of their ids: a row is the difference at its ends
        ids, order = torch.sort(s["ids"])
        edge = torch.searchsorted(ids, torch.arange(case["V"] + 1, device="cuda"))
        out = torch.empty(case["V"], case["D"], device="cuda", dtype=torch.float64)
        for c in range(0, case["D"], 512):
            run_ = torch.cumsum(s["grad_out"][order, c:c + 512].double(), 0)
            run_ = torch.cat((torch.zeros_like(run_[:1]), run_))
            out[:, c:c + 512] = (run_[edge[1:]] - run_[edge[:-1]]) * case["scale"]
        return out
    if op == "linear":
        x, n = s["x"].double(), []
        top = x.abs().max(1).values
        step = torch.where(top > 0, top, torch.ones_like(top))
        for a in range(0, case["M"], 8192):
            b = slice(a, a + 8192)
            y = torch.matmul((127.0 * x[b] / step[b, None]).round(), s["qw"].double().t())
            n.append(torch.addcmul(s["bias"].double().expand_as(y) if s["bias"] is not None else torch.zeros_like(y), y, top[b, None] / 127.0 * s["sw"].double()))
        return torch.cat(n)
    accept = torch.zeros(case["B"], case["K"], device="cuda", dtype=torch.float64)
    for b in range(case["B"]):
        n = case["K"] if s["lens"] is None else int(s["lens"][b])
        t = float(s["temperature"][b])
        for j in range(n):
            row, x = s["target"][b, j].double(), int(s["draft_tokens"][b, j])
            if t <= 0:
                accept[b, j] = float(int(torch.nonzero(row == row.max())[0, 0]) == x)
                continue
            lp = row[x] / t - torch.logsumexp(row / t, 0)
            if s["draft"] is not None:
                d = s["draft"][b, j].double() / t
                lp = lp - (d[x] - torch.logsumexp(d, 0))
            accept[b, j] = torch.exp(lp.clamp_max(0.0))
    return {"tokens": None, "counts": None, "accept": accept}
