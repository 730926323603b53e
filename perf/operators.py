"""The operators of svl.ops, as cases: multi-axis rotary positions, attention with capped scores,
distance bias, document and prefix masks, and products with 4-bit weights.

`run` computes a case in elementary torch operations (32 bits; 64 for rotation angles), or, where
`own` is true, makes the calls a program makes of svl.ops.  `exact` is the definition in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def ops():
    at = os.path.join(ROOT, "seldon-vault-lite-rust_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from svl import ops as module

    return module


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ cases --


def rope_case(name, dtype, tokens, q_heads, k_heads, head_dim, pairs, arrangement, grid, far):
    c = dict(op="rope", dtype=dtype, tokens=tokens, q_heads=q_heads, k_heads=k_heads, head_dim=head_dim, pairs=pairs,
             arrangement=arrangement, grid=grid, far=far)
    return dict(c, name=name) if name else c


def attention_case(name, dtype, q_heads, kv_heads, head_dim, batch, shortest, longest, rows=0, cap=0.0, slopes=False,
                   causal=False, window=-1, prefix=0, doc=0, padding=0, lengths=1):
    """rows: queries of each sequence (0: as many as keys); doc: mean tokens of a document (0: no documents);
    padding: trailing keys of each sequence that belong to no document."""
    c = dict(op="attention", dtype=dtype, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch,
             shortest=shortest, longest=longest, rows=rows, cap=cap, slopes=slopes, causal=causal, window=window,
             prefix=prefix, doc=doc, padding=padding, lengths=lengths)
    return dict(c, name=name) if name else c


def linear_case(name, dtype, rows, n, k, group, zeros):
    c = dict(op="linear", dtype=dtype, rows=rows, n=n, k=k, group=group, zeros=zeros)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one 32-token query through a sliding layer's heads (4 query and 2 key heads of 256): the smallest call
        rope_case("rope_query", "f32", 32, 4, 2, 256, "128", "sections", 1, 0),
        # the patches of a batch of images, 16 heads of 72, height and width each over half of the head
        rope_case("rope_images", "f16", 10007, 16, 16, 72, "18,18", "split", 2, 0),
        # a long video: time, height and width take the pairs in turn, time runs on from a far position
        rope_case("rope_video", "bf16", 65536, 16, 4, 128, "24,20,20", "interleaved", 3, 1000000),
        # one 32-token query over the sliding layer's heads in FP32: latency
        attention_case("attn_query_f32", "f32", 4, 2, 256, 1, 32, 32, cap=50.0),
        # a packed batch of documents cut into chunks behind a shared prompt: each chunk sees itself and the prompt
        attention_case("attn_chunks", "f16", 4, 2, 256, 64, 64, 512, prefix=9, doc=120, padding=3),
        # a two-sided encoder with a distance bias instead of rotary positions, 12 heads of 64
        attention_case("attn_bias", "f16", 12, 12, 64, 16, 700, 2048, slopes=True),
        # a long prompt read in order behind a prefix that is seen whole (an image's soft tokens), capped scores
        attention_case("attn_prefix", "bf16", 16, 2, 128, 2, 6000, 8192, cap=30.0, causal=True, prefix=1100),
        # the last token of each sequence over a long cache: one row a head
        attention_case("attn_last", "bf16", 32, 8, 128, 8, 9000, 65536, rows=1, cap=50.0, causal=True),
        # a query's single row through the q, k and v projections, FP32 activations: latency
        linear_case("linear_query", "f32", 1, 2048, 512, 32, False),
        # a 32-token query through the per-layer-input table's projection
        linear_case("linear_table", "f16", 32, 12288, 512, 64, True),
        # single tokens through a large block's down projection
        linear_case("linear_large", "bf16", 1, 8192, 28672, 128, False),
        # a few tokens, odd sizes
        linear_case("linear_odd", "bf16", 11, 5003, 2080, 32, True),
    ]


def spread(rng, low, high):
    """A whole number spread evenly over the logarithm of low..high."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "linear"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "rope":
        axes = rng.randint(1, 4)
        head_dim = 2 * spread(rng, 16, 128)
        most = head_dim // 2 // axes
        pairs = [rng.randint(max(1, most // 2), most) for _ in range(axes)]
        k_heads = rng.randint(1, 8)
        q_heads = k_heads * rng.choice([1, 2, 4])
        tokens = spread(rng, 1, max(1, min(65536, 160000000 // ((q_heads + k_heads) * head_dim))))
        return rope_case(None, dtype, tokens, q_heads, k_heads, head_dim, ",".join(map(str, pairs)),
                         rng.choice(["split", "sections", "interleaved"]), axes, rng.choice([0, 0, 1000000]))
    if op == "linear":
        group = rng.choice([32, 64, 128])
        k = group * spread(rng, 2, 28672 // group)
        n = spread(rng, 64, max(65, min(12288, 200000000 // k)))
        return linear_case(None, dtype, spread(rng, 1, 48), n, k, group, rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4])
    head_dim = rng.choice([64, 72, 80, 96, 128, 128, 192, 256])
    batch = spread(rng, 1, 32)
    single = rng.random() < 0.4
    if dtype == "f32":
        longest = spread(rng, 16, 1024)
    elif single:
        longest = spread(rng, 64, min(65536, 2 ** 28 // (batch * kv_heads * head_dim)))
    else:
        longest = spread(rng, 16, 8192)
    if not single:
        longest = min(longest, int(math.sqrt(8e10 / (batch * q_heads * head_dim))))
    shortest = max(1, int(longest * rng.uniform(0.2, 1.0)))
    rows = rng.randint(1, min(4, shortest)) if single else 0
    padding = rng.choice([0, 0, min(5, shortest - rows)])
    return attention_case(None, dtype, q_heads, kv_heads, head_dim, batch, shortest, longest, rows=rows,
                          cap=rng.choice([0.0, 30.0, 50.0]), slopes=rng.random() < 0.4, causal=rng.random() < 0.5,
                          window=rng.choice([-1, -1, max(1, longest // 4)]),
                          prefix=rng.choice([0, 0, max(1, longest // 10)]),
                          doc=rng.choice([0, max(2, longest // 4)]), padding=padding,
                          lengths=rng.randrange(1000))


# -------------------------------------------- what a case fixes besides values --


def lengths_of(c):
    """(queries, keys) of each sequence."""
    r = random.Random(c["lengths"])
    keys = [r.randint(c["shortest"], c["longest"]) for _ in range(c["batch"])]
    return [min(c["rows"] or n, n) for n in keys], keys


def documents_of(c, keys):
    """The document of each key, packed; -1 for padding; None without documents or padding."""
    if not c["doc"] and not c["padding"]:
        return None
    r = random.Random(c["lengths"] + 1)
    out = []
    for n in keys:
        d, ids = 0, []
        while len(ids) < n:
            ids += [d] * (r.randint(max(1, c["doc"] // 2), max(1, c["doc"] * 3 // 2)) if c["doc"] else n)
            d += 1
        ids = ids[:n]
        if c["padding"]:
            ids[n - c["padding"]:] = [-1] * c["padding"]
        out += ids
    return out


def cumulative(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def slopes_of(c):
    """A geometric run of distance slopes, one a query head; None without a distance bias."""
    return [2.0 ** (-8.0 * (h + 1) / c["q_heads"]) for h in range(c["q_heads"])] if c["slopes"] else None


def query_documents(c, lq, lk, docs):
    """Queries of their own belong to the documents of the last keys before the padding; others are the keys' rows."""
    if docs is None:
        return None
    out, at = [], 0
    for a, b in zip(lq, lk):
        end = at + b - (c["padding"] if c["rows"] else 0)
        out += docs[end - a:end]
        at += b
    return out


# ---------------------------------------------------------------- prepare --


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * by).to(t)

    if case["op"] == "rope":
        n, hd = case["tokens"], case["head_dim"]
        axes = [int(p) for p in case["pairs"].split(",")]
        # the fused q, k rows of a projection; positions walk a grid (time slowest, width fastest)
        qk = normal(n, (case["q_heads"] + case["k_heads"]) * hd)
        side = max(1, int(round(n ** (1.0 / len(axes)))))
        at = torch.arange(n, device="cuda") + torch.randint(0, 64, (1,), device="cuda", generator=g)
        pos = []
        for a in range(len(axes)):
            walk = at // side ** (len(axes) - 1 - a)
            pos.append((walk if a == 0 else walk % side) + (case["far"] if a == 0 else 0))
        s = dict(case=case, qk=qk, positions=torch.stack(pos).to(torch.int32), out=torch.empty_like(qk),
                 theta=[10000.0] * len(axes), pairs=axes)
        if own:
            s["rope"] = ops().AxisRope(hd, axes, s["theta"], arrangement=case["arrangement"])
        return s
    if case["op"] == "linear":
        n, k, group = case["n"], case["k"], case["group"]
        codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
        scales = ((torch.rand(n, k // group, device="cuda", generator=g) + 0.5) * 0.01).to(torch.bfloat16)
        zeros = torch.randint(5, 11, scales.shape, device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
        s = dict(case=case, x=normal(case["rows"], k), codes=codes, scales=scales, zeros=zeros,
                 y=torch.empty(case["rows"], n, device="cuda", dtype=t))
        if own:
            s["weight"] = ops().Q4Weight.from_codes(codes.data_ptr(), scales.data_ptr(), n, k, group,
                                                    zeros=zeros.data_ptr() if zeros is not None else 0)
        return s
    hq, hk, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    lq, lk = lengths_of(case)
    cu_q, cu_k = cumulative(lq), cumulative(lk)
    docs = documents_of(case, lk)
    doc_q = query_documents(case, lq, lk, docs)
    slopes = slopes_of(case)
    if case["rows"]:  # queries of their own over a cache
        q, k, v = normal(cu_q[-1], hq * hd, by=2.0), normal(cu_k[-1], hk * hd), normal(cu_k[-1], hk * hd)
    else:  # the fused rows of a q, k, v projection
        qkv = normal(cu_k[-1], (hq + 2 * hk) * hd)
        qkv[:, :hq * hd] *= 2.0
        q, k, v = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hk) * hd], qkv[:, (hq + hk) * hd:]

    def on_gpu(x, kind):
        return None if x is None else torch.tensor(x, dtype=kind, device="cuda")

    s = dict(case=case, q=q, k=k, v=v, out=torch.empty(cu_q[-1], hq * hd, device="cuda", dtype=t),
             lse=torch.empty(cu_q[-1], hq, device="cuda"), cu_q=on_gpu(cu_q, torch.int64), cu_k=on_gpu(cu_k, torch.int64),
             doc_q=on_gpu(doc_q, torch.int32), doc_k=on_gpu(docs, torch.int32), slopes=on_gpu(slopes, torch.float32),
             max_q=max(lq), max_k=max(lk))
    if own:
        plan = ops().AttentionPlan(hq, hk, hd, cu_q, cu_k, dtype=case["dtype"], scale=hd ** -0.5, cap=case["cap"],
                                   causal=case["causal"], window=case["window"] if case["window"] >= 0 else None,
                                   prefix=[case["prefix"]] * case["batch"] if case["prefix"] else None, doc_q=doc_q,
                                   doc_k=docs, slopes=slopes)
        s["plan"] = plan
        s["workspace"] = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------- rope --


def frequencies(pairs, thetas, arrangement, device):
    """(axis, first dim, second dim, frequency in 64 bits) of every rotation pair."""
    n = sum(pairs)
    axis = torch.arange(len(pairs), device=device).repeat_interleave(torch.tensor(pairs, device=device), output_size=n)
    if arrangement == "split":
        start = torch.tensor([2 * x for x in cumulative(pairs)[:-1]], device=device)[axis]
        inside = torch.arange(n, device=device) - start // 2
        count = torch.tensor(pairs, device=device)[axis]
        theta = torch.tensor(thetas, dtype=torch.float64, device=device)[axis]
        return axis, start + inside, start + inside + count, theta ** (-inside.double() / count)
    p = torch.arange(n, device=device)
    if arrangement == "interleaved":
        # the j-th pair of axis a comes in round j, after the earlier axes of that round
        turn = p - torch.tensor(cumulative(pairs)[:-1], device=device)[axis]
        axis = axis[torch.argsort(turn * len(pairs) + axis)]
    return axis, p, p + n, thetas[0] ** (-p.double() / n)


def plain_rope(s):
    c = s["case"]
    axis, first, second, f = frequencies(s["pairs"], s["theta"], c["arrangement"], s["qk"].device)
    angle = s["positions"].double()[axis].T * f
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s["qk"].float().view(c["tokens"], -1, c["head_dim"])
    a, b = x[..., first], x[..., second]
    y = x.clone()
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y.view(c["tokens"], -1).to(s["qk"].dtype)


def own_rope(s):
    c, qk, out = s["case"], s["qk"], s["out"]
    width, ahead = qk.shape[1], c["q_heads"] * c["head_dim"] * qk.element_size()
    s["rope"].apply_device(c["dtype"], s["positions"].data_ptr(), c["tokens"], qk.data_ptr(), width, c["q_heads"],
                           out.data_ptr(), width, qk.data_ptr() + ahead, width, c["k_heads"], out.data_ptr() + ahead,
                           width, stream=stream())
    return out


# ----------------------------------------------------------------- linear --


def plain_linear(s):
    c = s["case"]
    w = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(c["n"], c["k"] // c["group"], c["group"]).float()
    w = (w - (s["zeros"].float()[..., None] if c["zeros"] else 8.0)) * s["scales"].float()[..., None]
    return (s["x"].float() @ w.view(c["n"], c["k"]).T).to(s["x"].dtype)


def own_linear(s):
    c = s["case"]
    s["weight"].linear_device(c["dtype"], s["x"].data_ptr(), c["k"], c["rows"], s["y"].data_ptr(), c["n"],
                              stream=stream())
    return s["y"]


# -------------------------------------------------------------- attention --


def plain_attention(s):
    c = s["case"]
    hq, hk, hd, b, mq, mk = c["q_heads"], c["kv_heads"], c["head_dim"], c["batch"], s["max_q"], s["max_k"]
    dev = s["q"].device
    i, j = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    lq, lk = s["cu_q"].diff(), s["cu_k"].diff()
    rows = (s["cu_q"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    cols = (s["cu_k"][:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][rows].float().view(b, mq, hk, hq // hk, hd).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, hd)
    k = s["k"][cols].float().view(b, mk, hk, hd).permute(0, 2, 3, 1)
    v = s["v"][cols].float().view(b, mk, hk, hd).permute(0, 2, 1, 3)
    t = (q @ k).view(b, hk, hq // hk, mq, mk).mul_(hd ** -0.5)
    if c["cap"]:
        t = t.div_(c["cap"]).tanh_().mul_(c["cap"])
    place = i + (lk - lq)[:, None]
    gap = place[:, :, None] - j
    if c["slopes"]:
        t = t.sub_(s["slopes"].view(hk, -1, 1, 1) * gap.abs().float()[:, None, None])
    seen = torch.ones_like(gap, dtype=torch.bool)
    if c["causal"]:
        seen &= gap >= 0
    if c["window"] >= 0:
        seen &= gap.abs() <= c["window"]
    if s["doc_k"] is not None:
        dq, dk = s["doc_q"][rows], s["doc_k"][cols]
        seen &= dq[:, :, None] == dk[:, None]
    if c["prefix"]:
        seen |= j < c["prefix"]
    seen &= (j < lk[:, None])[:, None]
    if s["doc_k"] is not None:
        seen &= (dq >= 0)[:, :, None] & (dk >= 0)[:, None]
    t = t.masked_fill_(~seen[:, None, None], -math.inf)
    m = t.amax(-1, keepdim=True)
    e = t.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(b, hk, -1, mk) @ v).view(b, hq, mq, hd) / total.masked_fill(total == 0, 1.0).view(b, hq, mq, 1)
    lse = (m + total.log()).view(b, hq, mq)
    at = torch.arange(s["q"].shape[0], device=dev)
    of = torch.searchsorted(s["cu_q"], at, right=True) - 1
    at = at - s["cu_q"][of]
    return o[of, :, at].reshape(-1, hq * hd).to(s["q"].dtype), lse[of, :, at]


def own_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    s["plan"].run_device(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                         s["out"].data_ptr(), s["out"].stride(0), lse=s["lse"].data_ptr(),
                         workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), stream=stream())
    return s["out"], s["lse"]


def run(state):
    op = state["case"]["op"]
    if own:
        return own_rope(state) if op == "rope" else own_linear(state) if op == "linear" else own_attention(state)
    return plain_rope(state) if op == "rope" else plain_linear(state) if op == "linear" else plain_attention(state)


# ------------------------------------------------------------ work, exact --


def visible(c):
    """(query-key pairs that the masks leave, keys that some row sees), over the batch."""
    lq, lk = lengths_of(c)
    docs = documents_of(c, lk)
    doc_q = query_documents(c, lq, lk, docs)
    pairs, keys, at, row = 0, 0, 0, 0
    for a, b in zip(lq, lk):
        d = torch.tensor(docs[at:at + b]) if docs is not None else torch.zeros(b, dtype=torch.int64)
        dq = torch.tensor(doc_q[row:row + a]) if docs is not None else torch.zeros(a, dtype=torch.int64)
        live = torch.cat([torch.zeros(1, dtype=torch.int64), (d >= 0).long().cumsum(0)])
        p = torch.arange(a) + (b - a)
        low = (p - c["window"]).clamp(min=0) if c["window"] >= 0 else torch.zeros_like(p)
        high = p + 1 if c["causal"] else (p + c["window"] + 1).clamp(max=b) if c["window"] >= 0 else torch.full_like(p, b)
        if docs is not None:  # documents are runs: the row's own one starts and ends where its number does
            run = torch.where(d < 0, 1 << 30, d)
            low = torch.maximum(low, torch.searchsorted(run, dq))
            high = torch.minimum(high, torch.searchsorted(run, dq, right=True))
        f = min(c["prefix"], b)
        low, high = low.clamp(min=f), high.clamp(min=f)
        high = torch.where(dq < 0, low, torch.maximum(low, high))
        pairs += int((live[f] * (dq >= 0) + live[high] - live[low]).sum())
        edge = torch.zeros(b + 1, dtype=torch.int64).index_add_(0, low, torch.ones_like(low)).index_add_(0, high, -torch.ones_like(low))
        covered = edge.cumsum(0)[:b] > 0
        covered[:f] = True
        keys += int((covered & (d >= 0)).sum())
        at, row = at + b, row + a
    return pairs, keys


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        pairs = [int(p) for p in case["pairs"].split(",")]
        turned = case["tokens"] * (case["q_heads"] + case["k_heads"]) * sum(pairs)
        return {"bytes": 2 * n * size + 4 * len(pairs) * case["tokens"], "flops": 6 * turned}
    if case["op"] == "linear":
        n, k, m, groups = case["n"], case["k"], case["rows"], case["k"] // case["group"]
        return {"bytes": n * k // 2 + n * groups * (3 if case["zeros"] else 2) + m * (n + k) * size, "flops": 2 * m * n * k}
    lq, lk = lengths_of(case)
    hq, hk, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    pairs, keys = visible(case)
    return {"bytes": (2 * sum(lq) * hq + 2 * keys * hk) * hd * size + 4 * sum(lq) * hq, "flops": 4 * hd * hq * pairs}


def exact_attention(c, s):
    hq, hk, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
    lq, lk = lengths_of(c)
    out = torch.zeros(sum(lq), hq, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(lq), hq), -math.inf, dtype=torch.float64, device="cuda")
    slopes = slopes_of(c)
    row = col = 0
    for a, b in zip(lq, lk):
        p, j = torch.arange(b - a, b, device="cuda")[:, None], torch.arange(b, device="cuda")[None]
        hidden = torch.zeros(a, b, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= j > p
        if c["window"] >= 0:
            hidden |= (p - j).abs() > c["window"]
        if s["doc_k"] is not None:
            dq, dk = s["doc_q"][row:row + a, None], s["doc_k"][None, col:col + b]
            hidden |= dq != dk
        hidden &= j >= c["prefix"]
        if s["doc_k"] is not None:
            hidden |= (dq < 0) | (dk < 0)
        for h in range(hq):
            at = slice(h // (hq // hk) * hd, (h // (hq // hk) + 1) * hd)
            t = s["q"][row:row + a, h * hd:(h + 1) * hd].double() @ s["k"][col:col + b, at].double().T / math.sqrt(hd)
            if c["cap"]:
                t = torch.tanh(t / c["cap"]) * c["cap"]
            if slopes:
                t = t - slopes[h] * (p - j).abs()
            t = torch.where(hidden, -math.inf, t)
            z = torch.logsumexp(t, 1)
            w = torch.where(hidden, 0.0, torch.exp(t - z.clamp(min=-1e300)[:, None]))
            out[row:row + a, h], lse[row:row + a, h] = w @ s["v"][col:col + b, at].double(), z
        row, col = row + a, col + b
    return out.view(-1, hq * hd), lse


def exact_rope(c, s):
    hd, pairs = c["head_dim"], s["pairs"]
    y = s["qk"].double().clone().view(c["tokens"], -1, hd)
    x, total, turn, start = s["qk"].double().view(c["tokens"], -1, hd), sum(pairs), [], 0
    if c["arrangement"] == "split":
        for a, n in enumerate(pairs):
            turn += [(a, start + p, start + p + n, s["theta"][a] ** (-p / n)) for p in range(n)]
            start += 2 * n
    else:
        order = [a for a, n in enumerate(pairs) for _ in range(n)]
        if c["arrangement"] == "interleaved":
            order = [a for r in range(max(pairs)) for a, n in enumerate(pairs) if r < n]
        turn = [(a, p, p + total, s["theta"][0] ** (-p / total)) for p, a in enumerate(order)]
    for a, d, e, f in turn:
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"][a].double() * f)[:, None]
        z = torch.complex(x[..., d], x[..., e]) * z
        y[..., d], y[..., e] = z.real, z.imag
    return y.view(c["tokens"], -1)


def exact(case, seed):
    global own
    kept, own = own, False  # inputs alone: no plan
    s = prepare(case, seed)
    own = kept
    if case["op"] == "rope":
        return exact_rope(case, s)
    if case["op"] == "attention":
        return exact_attention(case, s)
    x, parts = s["x"].double(), []
    for at in range(0, case["n"], 1024):
        codes = s["codes"][at:at + 1024].long()
        w = torch.empty(codes.shape[0], case["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = codes % 16, codes // 16
        z = s["zeros"][at:at + 1024].double() if case["zeros"] else torch.full_like(s["scales"][at:at + 1024], 8).double()
        w -= z.repeat_interleave(case["group"], 1)
        w *= s["scales"][at:at + 1024].double().repeat_interleave(case["group"], 1)
        parts.append(x @ w.T)
    return torch.cat(parts, 1)
