"""The operators of a training step on packed documents, measured one by one: the embedding lookup whose gradient
is summed by sorted tokens, causal attention over documents of different lengths in one launch, and the vocabulary
projection with its cross entropy, which never holds the logits.

Widths, head counts and vocabularies are those of ``mist_b200/configs/model``, of ``bench.py`` and of the tests.  A
case is a dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` is the call: the
operators' plain form in fp32, or, where ``own`` is set, the framework's.
"""
import math
import random

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # ---- embedding: out = scale * wte[id] (+ wpe[position]); both tables' gradients
        # the benchmark's model (GPT-3 2.7B) at its micro batch: 8 x 2048 tokens, learned positions that restart
        # with every document; synthetic ids, uniform over the vocabulary
        dict(name="embed_gpt_2.7b_documents", op="embedding", tokens=16384, hidden=2560, vocab=50304, positions=2048,
             docs=11, ids="uniform", scale=1.0, backward=True),
        # a rotary model (no position table) on ids with the frequencies of text, scaled by sqrt(hidden)
        dict(name="embed_llama_7b_text", op="embedding", tokens=8192, hidden=4096, vocab=32000, positions=0,
             docs=5, ids="text", scale=64.0, backward=True),
        # a small odd batch, half of it the padding token: launches decide, one row takes most of the sum
        dict(name="embed_small_padded", op="embedding", tokens=333, hidden=512, vocab=1000, positions=128,
             docs=4, ids="padded", scale=1.0, backward=True),
        # ---- attention over packed documents
        # grouped-query training step of a 7B-width model: 16384 tokens of documents from tens to thousands of tokens
        dict(name="attn_llama_7b_documents", op="attention", tokens=16384, docs=14, longest=4096, heads=32, kv_heads=8,
             head_dim=128, causal=True, backward=True),
        # the benchmark's heads (32 of 80) on many short documents
        dict(name="attn_gpt_2.7b_short_docs", op="attention", tokens=8192, docs=61, longest=512, heads=32, kv_heads=32,
             head_dim=80, causal=True, backward=True),
        # whole prompts of a serving batch, forward only: ragged lengths, grouped heads
        dict(name="attn_prompts_forward", op="attention", tokens=6007, docs=7, longest=2048, heads=16, kv_heads=4,
             head_dim=128, causal=True, backward=False),
        # a handful of prompts of a few tokens, forward only: the latency of the smallest call
        dict(name="attn_few_tokens_forward", op="attention", tokens=93, docs=5, longest=40, heads=16, kv_heads=16,
             head_dim=64, causal=True, backward=False),
        # bidirectional encoder (masked-LM training) on packed sentences
        dict(name="attn_bert_sentences", op="attention", tokens=4099, docs=19, longest=512, heads=16, kv_heads=16,
             head_dim=128, causal=False, backward=True),
        # ---- vocabulary projection and cross entropy, logits never held
        # the benchmark's head: 8192 tokens of 2560, vocabulary 50304; the largest case
        dict(name="loss_gpt_2.7b", op="loss", tokens=8192, hidden=2560, vocab=50304, bias=False, ignored=0.0, backward=True),
        # masked-LM head: vocabulary bias, 15 % of the positions carry a label
        dict(name="loss_bert_masked", op="loss", tokens=4096, hidden=2048, vocab=50304, bias=True, ignored=0.85,
             backward=True),
        # perplexity of a text, forward only, odd number of tokens
        dict(name="loss_llama_7b_evaluation", op="loss", tokens=2047, hidden=4096, vocab=32000, bias=False, ignored=0.0,
             backward=False),
        # a first run of a tiny model: an odd vocabulary, few tokens
        dict(name="loss_small", op="loss", tokens=77, hidden=512, vocab=1003, bias=False, ignored=0.1, backward=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above, at most half the largest listed one's work."""
    most = 0.5 * max(_cost(c) for c in listed())
    op = rng.choice(["embedding", "attention", "attention", "loss", "loss"])
    while True:
        if op == "embedding":
            c = dict(op=op, tokens=_log_int(rng, 1, 30000), hidden=8 * _log_int(rng, 16, 512), vocab=_log_int(rng, 100, 100000),
                     positions=rng.choice([0, 0, 512, 2048]), docs=rng.randint(1, 20), ids=rng.choice(["uniform", "text", "padded"]),
                     scale=rng.choice([1.0, 0.5, 22.6]), backward=rng.random() < 0.8)
        elif op == "attention":
            longest, kv = _log_int(rng, 8, 4096), rng.choice([1, 2, 4, 8, 16])
            c = dict(op=op, docs=_log_int(rng, 1, 64), longest=longest, heads=kv * rng.choice([1, 1, 2, 4]), kv_heads=kv,
                     head_dim=rng.choice([32, 64, 80, 96, 128]), causal=rng.random() < 0.75, backward=rng.random() < 0.6)
            c["tokens"] = max(1, int(c["docs"] * longest * rng.uniform(0.2, 0.7)))
            if c["tokens"] > 16384 or c["docs"] * longest ** 2 * c["heads"] > 3e9:
                continue
        else:
            c = dict(op=op, tokens=_log_int(rng, 1, 8192), hidden=8 * _log_int(rng, 16, 512), vocab=_log_int(rng, 200, 50304),
                     bias=rng.random() < 0.4, ignored=rng.choice([0.0, 0.1, 0.85]), backward=rng.random() < 0.7)
        if _cost(c) <= most:
            return c


def _lengths(c):
    """Lengths of the case's documents: uneven, at most ``longest``, one of them a single token and (of many) one
    empty; their sum is the case's number of tokens."""
    n, total = c["docs"], c["tokens"]
    longest = c.get("longest") or min(c.get("positions") or total, total)
    r = random.Random(n * 100003 + total)
    share = [math.exp(r.uniform(0.0, 3.0)) for _ in range(n)]
    lens = [min(longest, int(s / sum(share) * total)) for s in share]
    if n >= 4:
        lens[1] = 1
    if n >= 10:
        lens[n // 2] = 0
    rest, i = total - sum(lens), 0
    while rest > 0:                                  # what is left goes to the first documents that have room
        if i >= n:
            lens.append(0)
            n += 1
        if n <= 4 or i not in (1, len(share) // 2):
            more = min(rest, longest - lens[i])
            lens[i] += more
            rest -= more
        i += 1
    return lens


def _visible(c):
    """(query, key) pairs that attention computes."""
    return sum(n * (n + 1) // 2 if c["causal"] else n * n for n in _lengths(c))


def work(case):
    c = case
    t, both = c["tokens"], c["backward"]
    if c["op"] == "embedding":
        h = c["hidden"]
        used = min(c["vocab"], t) if c["ids"] == "uniform" else min(c["vocab"], t) // 4 + 1
        pos = min(c["positions"], t) * h * 2 if c["positions"] else 0
        fwd = used * h * 2 + pos + t * h * 2 + t * 8
        bwd = t * h * 2 + c["vocab"] * h * 2 + c["positions"] * h * 2 + t * 8
        return {"bytes": fwd + (bwd if both else 0), "flops": 2 * t * h * (2 if both else 1)}
    if c["op"] == "attention":
        h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
        q, kv = t * h * d * 2, t * hk * d * 2
        io = 2 * q + 2 * kv + ((3 * q + 2 * kv) + q + 2 * kv if both else 0)
        return {"bytes": io, "flops": 4 * d * h * _visible(c) * (3.5 if both else 1)}
    h, v = c["hidden"], c["vocab"]
    io = (t * h + v * h) * 2 + t * 12 + ((t * h + v * h) * 2 * 2 + t * 4 if both else 0)
    return {"bytes": io, "flops": 2 * t * h * v * (3 if both else 1)}


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


# --------------------------------------------------------------------------------------- inputs
def _ids(c, gen):
    t, v = c["tokens"], c["vocab"]
    if c["ids"] == "text":                            # frequency about 1 / rank, ranks spread over the vocabulary
        u = torch.rand(t, generator=gen, device=DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(v + 1.0)) - 1).long().clamp_(0, v - 1)
        return torch.randperm(v, generator=gen, device=DEV)[rank]
    ids = torch.randint(0, v, (t,), generator=gen, device=DEV)
    if c["ids"] == "padded":
        ids = torch.where(torch.rand(t, generator=gen, device=DEV) < 0.5, torch.zeros_like(ids), ids)
    return ids


def _offsets(c):
    lens = _lengths(c)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return lens, torch.tensor(cu, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(torch.bfloat16)

    t, s = c["tokens"], {"case": c}
    if c["op"] == "embedding":
        lens, cu = _offsets(c)
        seg = torch.repeat_interleave(torch.tensor(lens, device=DEV))
        s["ids"] = _ids(c, gen)[None]
        s["wte"] = normal(c["vocab"], c["hidden"], std=0.02).requires_grad_(c["backward"])
        s["pos"] = s["wpe"] = None
        if c["positions"]:
            s["pos"] = (torch.arange(t, device=DEV) - cu[:-1].long()[seg])[None]
            s["wpe"] = normal(c["positions"], c["hidden"], std=0.02).requires_grad_(c["backward"])
        s["dout"] = normal(1, t, c["hidden"]) if c["backward"] else None
    elif c["op"] == "attention":
        # a projection's output: all q heads, then all k heads, then all v heads of a token
        h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
        s["lens"], s["cu"] = _offsets(c)
        s["qkv"] = normal(1, t, h + 2 * hk, d).requires_grad_(c["backward"])
        s["dout"] = normal(1, t, h, d) if c["backward"] else None
    else:
        v = c["vocab"]
        s["x"] = normal(t, c["hidden"]).requires_grad_(c["backward"])
        # logits of a few units, as a trained head gives
        s["weight"] = normal(v, c["hidden"], std=2.0 / math.sqrt(c["hidden"])).requires_grad_(c["backward"])
        s["bias"] = normal(v).requires_grad_(c["backward"]) if c["bias"] else None
        labels = torch.randint(0, v, (t,), generator=gen, device=DEV)
        off = torch.rand(t, generator=gen, device=DEV) < c["ignored"]
        s["labels"] = torch.where(off, torch.full_like(labels, -100), labels)
        s["dloss"] = (0.5 + torch.rand(t, generator=gen, device=DEV)) / t if c["backward"] else None
    return s


# ------------------------------------------------------------------------------- the operators
def run(state):
    c = state["case"]
    if own:
        return {"embedding": _own_embedding, "attention": _own_attention, "loss": _own_loss}[c["op"]](state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "attention": _plain_attention, "loss": _plain_loss}[c["op"]](state)


def _own_embedding(s):
    from mist_b200.ops import functional as F
    c, wte, wpe = s["case"], s["wte"], s["wpe"]
    out = F.embedding(s["ids"], wte, wpe, scale=c["scale"], position_ids=s["pos"])
    if not c["backward"]:
        return out
    return (out, *torch.autograd.grad(out, (wte,) if wpe is None else (wte, wpe), s["dout"]))


def _plain_embedding(s):
    c, ids, wte, wpe = s["case"], s["ids"][0], s["wte"], s["wpe"]
    out = wte.float()[ids] * c["scale"]
    if wpe is not None:
        out = out + wpe.float()[s["pos"][0]]
    out = out.to(wte.dtype)[None]
    if not c["backward"]:
        return out
    g = s["dout"][0].float()
    grads = [torch.zeros(wte.shape, device=DEV).index_add_(0, ids, g * c["scale"]).to(wte.dtype)]
    if wpe is not None:
        grads.append(torch.zeros(wpe.shape, device=DEV).index_add_(0, s["pos"][0], g).to(wpe.dtype))
    return (out, *grads)


def _own_attention(s):
    from mist_b200.ops import functional as F
    c, qkv = s["case"], s["qkv"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    scale = 1.0 / math.sqrt(d)
    if c["backward"]:
        out = F.attention_projected(qkv, hk, scale, c["causal"], packed=F.PackedSequences(s["cu"], c["tokens"]))
        return out, torch.autograd.grad(out, qkv, s["dout"])[0]
    q, k, v = qkv[0, :, :h], qkv[0, :, h:h + hk], qkv[0, :, h + hk:]
    return F.attention_varlen(q, k, v, s["cu"], scale=scale, causal=c["causal"])[None]


def _plain_attention(s):
    c, t = s["case"], s["case"]["tokens"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    scale, first, end = 1.0 / math.sqrt(d), s["cu"][:-1].long(), s["cu"][1:].long()
    longest = max(s["lens"])
    at = first[:, None] + torch.arange(longest, device=DEV)               # [documents, longest]
    real = at < end[:, None]
    at = at.clamp(max=t - 1)
    seg = torch.searchsorted(end, torch.arange(t, device=DEV), right=True)
    place = seg * longest + torch.arange(t, device=DEV) - first[seg]      # of every token in the padded layout

    def padded(x):
        return x.float()[at] * real[..., None, None]

    def packed(x):
        return x.reshape(-1, *x.shape[2:])[place]

    qkv = s["qkv"][0]
    n = len(s["lens"])
    q = padded(qkv[:, :h]).view(n, longest, hk, h // hk, d)
    k, v = padded(qkv[:, h:h + hk]), padded(qkv[:, h + hk:])
    hide = ~(real[:, None, :] & real[:, :, None])
    if c["causal"]:
        hide = hide | torch.ones(longest, longest, dtype=torch.bool, device=DEV).triu(1)
    p = torch.einsum("nqkgd,njkd->nkgqj", q, k).mul_(scale)
    p.masked_fill_(hide[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    out = packed(torch.einsum("nkgqj,njkd->nqkgd", p, v).reshape(n, longest, h, d)).to(qkv.dtype)[None]
    if not c["backward"]:
        return out
    g = padded(s["dout"][0]).view(n, longest, hk, h // hk, d)
    dv = torch.einsum("nkgqj,nqkgd->njkd", p, g)
    ds = torch.einsum("nqkgd,njkd->nkgqj", g, v)
    ds.sub_((p * ds).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.einsum("nkgqj,njkd->nqkgd", ds, k).reshape(n, longest, h, d)
    dk = torch.einsum("nkgqj,nqkgd->njkd", ds, q)
    return out, torch.cat([packed(dq), packed(dk), packed(dv)], 1).to(qkv.dtype)[None]


def _own_loss(s):
    from mist_b200.ops import functional as F
    x, weight, bias = s["x"], s["weight"], s["bias"]
    loss = F.linear_cross_entropy(x, weight, s["labels"], bias)
    if s["dloss"] is None:
        return loss
    return (loss, *torch.autograd.grad(loss, (x, weight) if bias is None else (x, weight, bias), s["dloss"]))


def _plain_loss(s):
    x, weight, bias, labels = s["x"].float(), s["weight"].float(), s["bias"], s["labels"]
    logits = x @ weight.t()
    if bias is not None:
        logits += bias.float()
    kept = labels != -100
    lab = labels.clamp(min=0)[:, None]
    top = logits.amax(-1, keepdim=True)
    target = logits.gather(1, lab)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    loss = torch.where(kept, (total.log() + top - target)[:, 0], torch.zeros_like(total[:, 0]))
    if s["dloss"] is None:
        return loss
    p.div_(total)
    p.scatter_add_(1, lab, torch.full_like(total, -1.0))
    p.mul_((s["dloss"] * kept)[:, None])
    grads = [(p @ weight).to(s["x"].dtype), (p.t() @ x).to(s["weight"].dtype)]
    if bias is not None:
        grads.append(p.sum(0).to(bias.dtype))
    return (loss, *grads)


# ------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    both = c["backward"]

    def wide(x):
        return None if x is None else x.detach().double().requires_grad_(both)

    if c["op"] == "embedding":
        wte, wpe = wide(s["wte"]), wide(s["wpe"])
        out = torch.nn.functional.embedding(s["ids"], wte) * c["scale"]
        if wpe is not None:
            out = out + torch.nn.functional.embedding(s["pos"], wpe)
        leaves, dout = [x for x in (wte, wpe) if x is not None], s["dout"]
    elif c["op"] == "attention":
        h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
        qkv, outs, first = wide(s["qkv"]), [], 0
        for n in s["lens"]:                           # one document and one key / value head at a time
            x = qkv[0, first:first + n]
            first += n
            heads = []
            for j in range(hk):
                q = x[:, j * (h // hk):(j + 1) * (h // hk)].transpose(0, 1)
                scores = q @ x[:, h + j].t() / math.sqrt(d)
                if c["causal"]:
                    scores = scores + torch.full((n, n), -math.inf, dtype=torch.float64, device=DEV).triu(1)
                heads.append(torch.softmax(scores, -1) @ x[:, h + hk + j])
            outs.append(torch.cat(heads).transpose(0, 1))
        out = torch.cat(outs)[None]
        leaves, dout = [qkv], s["dout"]
    else:
        x, weight, bias = wide(s["x"]), wide(s["weight"]), wide(s["bias"])
        logits = torch.nn.functional.linear(x, weight, bias)
        kept = s["labels"] >= 0
        picked = logits.gather(1, s["labels"].clamp(min=0)[:, None])[:, 0]
        out = (torch.logsumexp(logits, -1) - picked) * kept
        leaves, dout = [x for x in (x, weight, bias) if x is not None], s["dloss"]
    if not both:
        return out
    grads = torch.autograd.grad(out, leaves, dout.double())
    return (out.detach(), *grads)
