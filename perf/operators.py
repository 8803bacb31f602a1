"""The operators around the text tower and the training step that are measured by themselves: token lookup and its gradient,
causal attention over packed prompts (forward, and forward + backward), and clipping by the global gradient norm.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, with
`own`, through the framework's entry points.  `exact` gives the same outputs from the definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}


def listed():
    return [
        # the text tower's lookup for a single prompt (77 tokens, vocabulary and width of the 1024-wide tower): pure latency
        dict(name="lookup, one prompt", op="lookup", tokens=77, vocab=49408, width=1024, ids="prompts", table="fp32", out="bf16",
             scale=1.0),
        # a packed corpus of prompts through a bf16 table, scaled by sqrt(width): bandwidth
        dict(name="lookup, packed corpus", op="lookup", tokens=50021, vocab=49408, width=1024, ids="zipf", table="bf16", out="bf16",
             scale=32.0),
        # a training batch of 32 padded prompts: most positions hold the padding token, one row of the table takes them all
        dict(name="lookup gradient, 32 prompts", op="lookup_grad", tokens=2464, vocab=49408, width=1024, ids="prompts", grad="bf16",
             scale=1.0, padding=-1),
        # a packed corpus: many rows with few tokens, a few rows with thousands
        dict(name="lookup gradient, corpus", op="lookup_grad", tokens=131071, vocab=49408, width=1024, ids="zipf", grad="bf16",
             scale=32.0, padding=-1),
        # class embeddings and learned tables of odd width, with a padding row that takes no gradient
        dict(name="lookup gradient, odd table", op="lookup_grad", tokens=5003, vocab=1003, width=333, ids="uniform", grad="fp32",
             scale=1.0, padding=0),
        # one prompt of the text tower: pure latency
        dict(name="attention, one prompt", op="attention", seqs=1, low=77, high=77, lens=1, pad=0, heads=16, kv_heads=16, d=64,
             train=False),
        # a batch of ragged prompts, packed instead of padded, in a buffer with some rows behind the last one
        dict(name="attention, 32 prompts", op="attention", seqs=32, low=5, high=77, lens=2, pad=51, heads=16, kv_heads=16, d=64,
             train=False),
        # long ragged prompts with grouped heads
        dict(name="attention, long grouped", op="attention", seqs=4, low=1500, high=8192, lens=3, pad=0, heads=32, kv_heads=8, d=128,
             train=False),
        # a training batch of ragged prompts
        dict(name="attention training, 64 prompts", op="attention", seqs=64, low=5, high=77, lens=4, pad=0, heads=16, kv_heads=16,
             d=64, train=True),
        # training on long ragged texts with grouped heads
        dict(name="attention training, long", op="attention", seqs=5, low=300, high=4096, lens=5, pad=0, heads=16, kv_heads=4, d=64,
             train=True),
        # every gradient of the ControlNet's training step at the SD-2.1 geometry, the norm above the limit
        dict(name="clip, ControlNet", op="clip", tensors="controlnet", dtype="fp32", gap=128, active=True, sizes=0, count=0, most=0),
        # a fine-tuned handful of small tensors whose norm stays below the limit: nothing to scale, pure latency
        dict(name="clip, norms and biases", op="clip", tensors="random", dtype="fp32", gap=128, active=False, sizes=7, count=40,
             most=1280),
    ]


def spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), cost(c))
    while True:
        op = rng.choice(["lookup", "lookup_grad", "lookup_grad", "attention", "attention", "attention", "clip"])
        width = spread(rng, 8, 256) * 8 if rng.random() < 0.6 else spread(rng, 64, 2048)
        c = dict(op=op)
        if op == "lookup":
            c.update(tokens=spread(rng, 1, 65536), vocab=spread(rng, 100, 131072), width=width, ids=rng.choice(["uniform", "zipf"]),
                     table=rng.choice(["fp32", "bf16"]), out=rng.choice(["bf16", "bf16", "fp32"]), scale=rng.choice([1.0, 22.6, 32.0]))
        elif op == "lookup_grad":
            c.update(tokens=spread(rng, 1, 131071), vocab=spread(rng, 100, 131072), width=width,
                     ids=rng.choice(["uniform", "zipf", "one"]), grad=rng.choice(["bf16", "bf16", "fp32"]),
                     scale=rng.choice([1.0, 22.6, 32.0]), padding=rng.choice([-1, 0]))
        elif op == "attention":
            high = spread(rng, 1, 8192)
            kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
            c.update(seqs=spread(rng, 1, 64), low=spread(rng, 1, high), high=high, lens=rng.randrange(1 << 20),
                     pad=rng.choice([0, 0, 37, 130]), heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads,
                     d=rng.choice([64, 128]), train=rng.random() < 0.5)
            # the plain form holds every score of a padded batch at once
            if c["seqs"] * c["heads"] * high * high > (3 << 30 if c["train"] else 8 << 30):
                continue
        else:
            c.update(tensors="random", dtype=rng.choice(["fp32", "fp32", "bf16"]), gap=rng.choice([1, 128]),
                     active=rng.random() < 0.6, sizes=rng.randrange(1 << 20), count=spread(rng, 1, 400), most=spread(rng, 64, 1 << 24))
        if cost(c) <= most[op]:
            return c


# ------------------------------------------------------------------ sizes that follow from a case
def lengths(case):
    """The sequences' lengths: log-uniform in [low, high], one of them (at a random place) the longest."""
    rng = random.Random(case["lens"])
    got = [spread(rng, case["low"], case["high"]) for _ in range(case["seqs"])]
    got[rng.randrange(len(got))] = case["high"]
    return got


def controlnet_sizes():
    """The parameters' sizes of a ControlNet at the SD-2.1 geometry: (320, 640, 1280, 1280) channels, two residual blocks a
    level, attention with 1024-wide context on the first three levels, conditioning channels (64, 128, 128, 256)."""
    sizes, emb, ctx, prev = [], 1280, 1024, 320

    def layer(cin, cout, k=1, bias=True):
        sizes.extend([cin * cout * k * k] + [cout] * bias)

    def norm(c):
        sizes.extend([c, c])

    def resnet(cin, cout):
        norm(cin), layer(cin, cout, 3), layer(emb, cout), norm(cout), layer(cout, cout, 3)
        if cin != cout:
            layer(cin, cout)

    def transformer(c):
        norm(c), layer(c, c)
        for kv in (c, ctx):
            layer(c, c, bias=False), layer(kv, c, bias=False), layer(kv, c, bias=False), layer(c, c)
        layer(c, 8 * c), layer(4 * c, c), norm(c), norm(c), norm(c), layer(c, c)

    layer(4, 320, 3), layer(320, emb), layer(emb, emb)
    cond = [64, 128, 128, 256]
    layer(1, cond[0], 3)
    for a, b in zip(cond, cond[1:]):
        layer(a, a, 3), layer(a, b, 3)
    layer(cond[-1], 320, 3), layer(320, 320)
    for level, c in enumerate([320, 640, 1280, 1280]):
        for _ in range(2):
            resnet(prev, c)
            if level < 3:
                transformer(c)
            layer(c, c)
            prev = c
        if level < 3:
            layer(c, c, 3), layer(c, c)
    resnet(1280, 1280), transformer(1280), resnet(1280, 1280), layer(1280, 1280)
    return sizes


def clip_sizes(case):
    if case["tensors"] == "controlnet":
        return controlnet_sizes()
    rng = random.Random(case["sizes"])
    sizes = [spread(rng, 1, case["most"]) for _ in range(case["count"])]
    while sum(sizes) > 1 << 28:  # at most the ControlNet's order of size in all
        sizes.pop()
    return sizes


def work(case):
    op = case["op"]
    if op == "lookup":
        rows = min(case["tokens"], case["vocab"])
        n = case["tokens"] * case["width"]
        return {"bytes": 8 * case["tokens"] + rows * case["width"] * SIZE[case["table"]] + n * SIZE[case["out"]], "flops": n}
    if op == "lookup_grad":
        n = case["tokens"] * case["width"]
        return {"bytes": 8 * case["tokens"] + n * SIZE[case["grad"]] + case["vocab"] * case["width"] * 4, "flops": 2 * n}
    if op == "attention":
        lens, h, kv, d = lengths(case), case["heads"], case["kv_heads"], case["d"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        rows = sum(lens)
        q, k = rows * h * d * 2, rows * kv * d * 2
        # two products forward; five backward (the scores again, dP, dQ, dK, dV) over the gradient, q, k, v and o
        return {"bytes": 2 * q + 2 * k + (3 * q + q + 4 * k if case["train"] else 0), "flops": (14 if case["train"] else 4) * d * h * pairs}
    n = sum(clip_sizes(case)) * SIZE[case["dtype"]]
    # a norm reads every gradient; scaling reads them again and writes them
    return {"bytes": n * (3 if case["active"] else 1), "flops": sum(clip_sizes(case)) * (3 if case["active"] else 2)}


def cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200)


# ------------------------------------------------------------------ inputs
def make_ids(case, gen):
    t, v = case["tokens"], case["vocab"]
    if case["ids"] == "uniform":
        return torch.randint(0, v, (t,), generator=gen, device="cuda")
    if case["ids"] == "one":  # three quarters of the positions hold one token
        ids = torch.randint(0, v, (t,), generator=gen, device="cuda")
        return torch.where(torch.rand(t, generator=gen, device="cuda") < 0.75, ids[0], ids)
    if case["ids"] == "zipf":  # the frequency of token r falls as 1 / r, as in text
        u = torch.rand(t, generator=gen, device="cuda", dtype=torch.float64)
        return (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)
    # prompts of 77: a start token, 3 to 30 words, then the end token to the end
    rows = -(-t // 77)
    ids = torch.randint(0, v - 2, (rows, 77), generator=gen, device="cuda")
    words = torch.randint(3, 31, (rows, 1), generator=gen, device="cuda")
    at = torch.arange(77, device="cuda")
    ids = torch.where(at > words, v - 1, ids)
    ids[:, 0] = v - 2
    return ids.reshape(-1)[:t].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    if op == "lookup":
        s["ids"] = make_ids(case, gen)
        s["weight"] = normal(case["vocab"], case["width"], dtype=DTYPES[case["table"]], scale=0.02)
    elif op == "lookup_grad":
        s["ids"] = make_ids(case, gen)
        s["dy"] = normal(case["tokens"], case["width"], dtype=DTYPES[case["grad"]], scale=1e-3)
    elif op == "attention":
        lens, h, kv, d = lengths(case), case["heads"], case["kv_heads"], case["d"]
        rows = sum(lens) + case["pad"]
        # one matrix from the fused projection; queries, keys and values are its columns
        qkv = normal(rows, (h + 2 * kv) * d, dtype=torch.bfloat16)
        qkv[:, :h * d] *= 2  # attention that has something to choose
        s["q"], s["k"], s["v"] = qkv[:, :h * d], qkv[:, h * d:(h + kv) * d], qkv[:, (h + kv) * d:]
        ends = [0]
        for n in lens:
            ends.append(ends[-1] + n)
        s["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["lens"] = torch.tensor(lens, device="cuda")
        s["longest"] = max(lens)
        if case["train"]:
            s["do"] = normal(rows, h * d, dtype=torch.bfloat16, scale=0.1)
    else:
        sizes, dt, gap = clip_sizes(case), DTYPES[case["dtype"]], case["gap"]
        starts, total = [], 0
        for n in sizes:  # gap 128: each tensor at an aligned place of its own; gap 1: packed end to end
            starts.append(total)
            total += -(-n // gap) * gap
        flat, out = torch.zeros(total, dtype=dt, device="cuda"), torch.zeros(total, dtype=dt, device="cuda")
        s["grads"] = [flat[a:a + n] for a, n in zip(starts, sizes)]
        for g in s["grads"]:
            g.copy_(normal(g.numel(), dtype=dt, scale=1e-2))
        norm = 1e-2 * math.sqrt(sum(sizes))
        s["limit"] = norm * (0.2 if case["active"] else 4.0)
        # an active limit scales into a second set of tensors, so that the next pass finds the same gradients
        s["outs"] = [out[a:a + n] for a, n in zip(starts, sizes)] if case["active"] else s["grads"]
        s["flat"] = out if case["active"] else flat
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["op"]
    if own:
        from ccnet_amd import ops
        if op == "lookup":
            return ops.embedding(s["ids"], s["weight"], scale=s["scale"], dtype=DTYPES[s["out"]])
        if op == "lookup_grad":
            return ops.embedding_grad(s["ids"], s["dy"], s["vocab"], scale=s["scale"],
                                      padding_idx=None if s["padding"] < 0 else s["padding"])
        if op == "attention":
            h, kv, d = s["heads"], s["kv_heads"], s["d"]
            if not s["train"]:
                return ops.attention_packed(s["q"], s["k"], s["v"], s["cu"], h, kv, d, d ** -0.5)
            o, lse = ops.attention_packed(s["q"], s["k"], s["v"], s["cu"], h, kv, d, d ** -0.5, with_lse=True)
            return (o,) + ops.attention_packed_bwd(s["q"], s["k"], s["v"], o, s["do"], lse, s["cu"], h, kv, d, d ** -0.5)
        norm = ops.clip_grad_norm(s["grads"], s["limit"], out=s["outs"] if s["active"] else None)
        return norm, s["flat"]
    if op == "lookup":
        return (s["weight"][s["ids"]].float() * s["scale"]).to(DTYPES[s["out"]])
    if op == "lookup_grad":
        grad = torch.zeros(s["vocab"], s["width"], dtype=torch.float64, device="cuda")  # long sums
        grad.index_add_(0, s["ids"], s["dy"].double())
        if s["padding"] >= 0:
            grad[s["padding"]] = 0
        return (grad * s["scale"]).float()
    if op == "attention":
        return plain_attention(s)
    total = torch.stack([g.float().square().sum() for g in s["grads"]]).sum()
    norm = total.sqrt()
    factor = (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * factor) for o, g in zip(s["outs"], s["grads"])]
    return norm, s["flat"]


def plain_attention(s):
    """The sequences as a padded batch [sequence, kv head, query head of the group, row, channel], in 32 bits."""
    longest, h, kv, d = s["longest"], s["heads"], s["kv_heads"], s["d"]
    at = torch.arange(longest, device="cuda")
    real = at < s["lens"][:, None]  # [sequence, row]
    total = s["q"].shape[0]
    rows = s["cu"][:-1, None].long() + at  # the packed row of each; one past the last for what is padding
    rows = torch.where(real, rows, total)
    scale = d ** -0.5

    def padded(x, heads):
        y = x[rows.clamp(max=total - 1)].float() * real[:, :, None]
        return y.unflatten(2, (heads, d)).permute(0, 2, 1, 3).unflatten(1, (kv, heads // kv)).contiguous()

    def packed(y, like):
        out = torch.zeros(total + 1, like.shape[1], dtype=torch.bfloat16, device="cuda")
        out[rows] = y.flatten(1, 2).permute(0, 2, 1, 3).flatten(2).to(torch.bfloat16)
        return out[:-1]

    q, k, v = padded(s["q"], h), padded(s["k"], kv), padded(s["v"], kv)
    p = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(at > at[:, None], -math.inf)  # key > query
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = packed(p @ v, s["q"])
    if not s["train"]:
        return o
    do = padded(s["do"], h)
    ds = do @ v.transpose(-1, -2)
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return o, packed(dq, s["q"]), packed(dk, s["k"]), packed(dv, s["v"])


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        return torch.index_select(s["weight"], 0, s["ids"]).double() * case["scale"]
    if op == "lookup_grad":
        # tokens in sorted order, a running sum down the rows, and differences of it at the ends of each run: columns in turn
        order = torch.argsort(s["ids"], stable=True)
        counts = torch.bincount(s["ids"], minlength=case["vocab"])
        ends = torch.cumsum(counts, 0)
        grad = torch.empty(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        for c in range(0, case["width"], 128):
            run_sum = torch.cumsum(s["dy"][:, c:c + 128].double()[order], 0)
            run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
            grad[:, c:c + 128] = run_sum[ends] - run_sum[ends - counts]
        if case["padding"] >= 0:
            grad[case["padding"]] = 0
        return grad * case["scale"]
    if op == "attention":
        h, kv, d = case["heads"], case["kv_heads"], case["d"]
        q, k, v = (s[x].double().requires_grad_(case["train"]) for x in "qkv")
        outs = [torch.zeros(s[x].shape, dtype=torch.float64, device="cuda") for x in ("qqkv" if case["train"] else "q")]
        first = 0
        for n in lengths(case):
            rows = slice(first, first + n)
            first += n
            future = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            for head in range(h):
                mine, shared = slice(head * d, head * d + d), slice(head // (h // kv) * d, head // (h // kv) * d + d)
                parts = [x[rows, c].detach().requires_grad_(case["train"]) for x, c in ((q, mine), (k, shared), (v, shared))]
                scores = (parts[0] @ parts[1].T / math.sqrt(d)).masked_fill(future, -math.inf)
                o = torch.softmax(scores, -1) @ parts[2]
                outs[0][rows, mine] = o.detach()
                if case["train"]:
                    got = torch.autograd.grad(o, parts, s["do"][rows, mine].double())
                    outs[1][rows, mine] = got[0]
                    outs[2][rows, shared] += got[1]
                    outs[3][rows, shared] += got[2]
        return tuple(outs) if case["train"] else outs[0]
    parts = [g.double() for g in s["grads"]]
    norm = math.sqrt(math.fsum(float((g * g).sum()) for g in parts))
    factor = min(1.0, s["limit"] / (norm + 1e-6))
    flat = s["flat"].double()
    for o, g in zip(s["outs"], parts):
        at = o.storage_offset()
        flat[at:at + o.numel()] = g * factor
    return torch.tensor(norm, dtype=torch.float64, device="cuda"), flat
