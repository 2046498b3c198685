"""Operators of the attention block over the paged KV cache, as a server uses them.

``append``   token runs enter the cache: RMS norm of the q and k heads, rotary positions of one or three axes,
             K and V rows into 256-position chunks (f16 or q8_0), q and gate out.
``prefill``  causal attention of ragged token runs over the cache that already holds them.
``shared``   one decode step of sequences that share long prefixes.

16 query heads, 4 key/value heads, 256 dimensions a head, rotation over the first 64 of them.
"""
import math

import torch

own = False

HEADS, KV_HEADS, DIM, CHUNK, PAIRS = 16, 4, 256, 256, 32
GROUP = HEADS // KV_HEADS
QKV = HEADS * 2 * DIM + 2 * KV_HEADS * DIM  # q | gate per head, then k, then v
Q8_ROW = DIM // 32 * 34  # q8_0 blocks {f16 d; int8 q[32]}
EPS = 1e-6


def listed():
    return [
        # one token of one sequence at the end of a 4096-token context: the latency of a batch-1 step
        {"name": "append_token", "op": "append", "runs": "4095+1", "axes": 1, "interleaved": True, "half": False, "q8": False},
        # a decode step of 32 sequences over the quantised cache
        {"name": "append_batch32_q8", "op": "append", "runs": "*32:511+1:97", "axes": 1, "interleaved": True, "half": False,
         "q8": True},
        # prompts with pictures, several requests packed into one pass
        {"name": "append_images", "op": "append", "runs": "0+733,129+1024,4001+17,0+61,255+2", "axes": 3,
         "interleaved": True, "half": True, "q8": False},
        # one long prompt with pictures, sections in contiguous order
        {"name": "append_prompt", "op": "append", "runs": "0+8192", "axes": 3, "interleaved": False, "half": True, "q8": False},
        # a run of a single token: the decode form
        {"name": "prefill_token", "op": "prefill", "runs": "4095+1", "window": 0, "sink": 0, "half": False, "q8": False},
        # the runtime's run of 64 tokens, deep into a long context
        {"name": "prefill_run64", "op": "prefill", "runs": "32704+64", "window": 0, "sink": 0, "half": False, "q8": False},
        # several requests of odd sizes in one pass, sliding window with sinks
        {"name": "prefill_ragged", "op": "prefill", "runs": "0+733,129+1024,4001+17,0+61,255+2,1500+301", "window": 1024,
         "sink": 4, "half": True, "q8": False},
        # one long prompt
        {"name": "prefill_prompt", "op": "prefill", "runs": "0+8192", "window": 0, "sink": 0, "half": True, "q8": False},
        # two samples of one short question
        {"name": "shared_pair", "op": "shared", "groups": "2*700", "tail": 40, "window": 0, "sink": 0, "half": False, "q8": False},
        # 32 users behind one system prompt
        {"name": "shared_batch32", "op": "shared", "groups": "32*4096", "tail": 256, "window": 0, "sink": 0, "half": True,
         "q8": False},
        # 32 questions about one long document
        {"name": "shared_document", "op": "shared", "groups": "32*32768", "tail": 512, "window": 0, "sink": 0, "half": False,
         "q8": False},
        # three prompts of odd lengths with their own users, quantised cache
        {"name": "shared_groups_q8", "op": "shared", "groups": "34*9001,5*20011,1*1357", "tail": 333, "window": 0, "sink": 0,
         "half": False, "q8": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "prefill", "shared"])
    half, q8 = rng.random() < 0.5, rng.random() < 0.3
    if op == "append":
        left, runs = _log(rng, 1, 8192), []
        while left > 0 and len(runs) < 12:
            n = _log(rng, 1, left)
            runs.append("%d+%d" % (_log(rng, 1, 6000) - 1, n))
            left -= n
        return {"op": op, "runs": ",".join(runs), "axes": rng.choice([1, 3]), "interleaved": rng.random() < 0.6, "half": half,
                "q8": q8}
    window = _log(rng, 16, 4096) if rng.random() < 0.3 else 0
    sink = rng.randint(0, 40) if window else 0
    if op == "prefill":
        left, runs = _log(rng, 1, 5000), []
        while left > 0 and len(runs) < 8:
            n = _log(rng, 1, left)
            runs.append("%d+%d" % (_log(rng, 1, 6000) - 1, n))
            left -= n
        return {"op": op, "runs": ",".join(runs), "window": window, "sink": sink, "half": half, "q8": q8}
    groups = ["%d*%d" % (_log(rng, 1, 40), _log(rng, 1, 24000)) for _ in range(rng.randint(1, 3))]
    return {"op": op, "groups": ",".join(groups[:1 if half else 3]), "tail": _log(rng, 1, 600), "window": window, "sink": sink,
            "half": half, "q8": q8}


# ---- the shapes behind a case -----------------------------------------------------------

def _runs(case):
    """[(positions already in the cache, tokens of the run)] of an append or prefill case."""
    text = case["runs"]
    if text.startswith("*"):  # "*n:ctx+len:step": n runs, each `step` positions further in
        n, run, step = text[1:].split(":")
        ctx, length = run.split("+")
        return [(int(ctx) + i * int(step), int(length)) for i in range(int(n))]
    return [tuple(int(v) for v in r.split("+")) for r in text.split(",")]


def _sequences(case):
    """(sequences per group, shared length per group, total length per sequence) of a shared case."""
    groups = [tuple(int(v) for v in g.split("*")) for g in case["groups"].split(",")]
    counts, shared, total = [g[0] for g in groups], [g[1] for g in groups], []
    for n, s in groups:
        for _ in range(n):
            total.append(s + 1 + (37 * len(total) + 11) % case["tail"])
    return counts, shared, total


def _attended(length, window, sink):
    """Positions that a query of context length `length` attends."""
    sink = min(sink, length)
    return length if window <= 0 or sink + window >= length else sink + window


def work(case):
    row = 2 * KV_HEADS * (Q8_ROW if case["q8"] else 2 * DIM)  # K and V bytes of a position
    value = 2 if case["half"] else 4
    if case["op"] == "append":
        n = sum(r for _, r in _runs(case))
        return {"bytes": n * (4 * QKV + 2 * HEADS * DIM * value + row + 4 * (case["axes"] + 2)) + 4 * (2 * DIM + PAIRS),
                "flops": n * ((HEADS + KV_HEADS) * DIM * 4 + (HEADS + KV_HEADS) * PAIRS * 6)}
    w, s = case["window"], case["sink"]
    if case["op"] == "prefill":
        runs = _runs(case)
        n = sum(r for _, r in runs)
        pairs = sum(_attended(c + t + 1, w, s) for c, r in runs for t in range(r))
        # positions of the cache that at least one token of the run attends
        keys = sum(c + r if w <= 0 else min(c + r, w + r + s) for c, r in runs)
    else:
        counts, shared, total = _sequences(case)
        n = len(total)
        pairs = sum(_attended(t, w, s) for t in total)
        keys, i = 0, 0
        for c, p in zip(counts, shared):
            tails = [t - p for t in total[i:i + c]]
            i += c
            keys += p if w <= 0 else min(p, w + s)
            keys += sum(t if w <= 0 else min(t, w + s) for t in tails)
    return {"bytes": keys * row + 3 * n * HEADS * DIM * value, "flops": pairs * HEADS * DIM * 4}


# ---- inputs -------------------------------------------------------------------------------

def _cache(lengths, q8, gen, fill):
    """A pool of chunks in shuffled order and each sequence's chunk numbers; `fill`: K rows of unit RMS, V normal."""
    chunks = [max(1, -(-n // CHUNK)) for n in lengths]
    perm = torch.randperm(sum(chunks), generator=gen).tolist()
    table = torch.zeros(len(lengths), max(chunks), dtype=torch.int64)
    at = 0
    for i, c in enumerate(chunks):
        table[i, :c] = torch.tensor(perm[at:at + c])
        at += c
    return _pool(at, q8, int(torch.randint(1 << 30, (1,), generator=gen)), fill), table


def _pool(chunks, q8, seed, fill):
    gen = torch.Generator("cuda").manual_seed(seed)
    if not q8:
        pool = torch.zeros(chunks, 2, KV_HEADS, CHUNK, DIM, dtype=torch.float16, device="cuda")
        if fill:
            pool.normal_(generator=gen)
        return pool
    pool = torch.zeros(chunks, 2, KV_HEADS, CHUNK, DIM // 32, 34, dtype=torch.uint8, device="cuda")
    if fill:
        q = torch.randint(-127, 128, pool.shape[:-1] + (32,), dtype=torch.int8, device="cuda", generator=gen)
        d = (0.6 + 0.8 * torch.rand(pool.shape[:-1] + (1,), device="cuda", generator=gen)) * (1.7 / 127)
        pool[..., 2:] = q.view(torch.uint8)
        pool[..., :2] = d.to(torch.float16).view(torch.uint8)
    return pool


def _addresses(pool, table):
    """The chunk table as the framework takes it: each chunk's address on the device."""
    return table.to("cuda") * (pool[0].numel() * pool.element_size()) + pool.data_ptr()


def _rotary(runs, axes):
    """Positions [axes, tokens]: text counts on; a picture keeps its time and spreads over rows and columns."""
    out = []
    for ctx, n in runs:
        picture = n // 2 if axes == 3 and n >= 24 else 0
        before, width, p = (n - picture) // 2, max(1, int(math.sqrt(picture) * 1.3)), ctx
        for t in range(n):
            if before <= t < before + picture:
                k = t - before
                out.append((p, p + k // width, p + k % width))
                if k == picture - 1:
                    p += max(width, k // width + 1)
            else:
                out.append((p, p, p))
                p += 1
    return torch.tensor(out, dtype=torch.int32).t()[:axes].contiguous()


def prepare(case, seed):
    gen = torch.Generator().manual_seed(int(seed))
    dev = torch.Generator("cuda").manual_seed(int(seed) + 1)
    kind = torch.float16 if case["half"] else torch.float32
    q8 = case["q8"]
    s = {"case": case, "kind": kind, "v_off": KV_HEADS * CHUNK * (Q8_ROW if q8 else 2 * DIM)}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "append":
        runs = _runs(case)
        n = sum(r for _, r in runs)
        s["pool"], s["table"] = _cache([c + r for c, r in runs], q8, gen, False)
        s["qkv"] = torch.randn(n, QKV, device="cuda", generator=dev) * (0.5 + torch.rand(n, 1, device="cuda", generator=dev))
        s["q_norm"], s["k_norm"] = (1 + 0.2 * torch.randn(DIM, device="cuda", generator=dev) for _ in range(2))
        s["freq"] = (1e7 ** (-torch.arange(PAIRS, dtype=torch.float64) / PAIRS)).to(torch.float32).cuda()
        s["rotary"] = _rotary(runs, case["axes"]).cuda()
        s["sections"] = (11, 11, 10) if case["axes"] == 3 else (PAIRS,)
        s["tok_seq"] = ints([i for i, (_, r) in enumerate(runs) for _ in range(r)])
        s["tok_pos"] = ints([c + t for c, r in runs for t in range(r)])
    else:
        if case["op"] == "prefill":
            runs = _runs(case)
            lengths, n = [c + r for c, r in runs], sum(r for _, r in runs)
            s["pool"], s["table"] = _cache(lengths, q8, gen, True)
            offsets = [0]
            for _, r in runs:
                offsets.append(offsets[-1] + r)
            s["run_off"], s["max_run"], s["max_len"] = ints(offsets), max(r for _, r in runs), max(lengths)
            s["seq_len"] = ints(lengths)
        else:
            counts, shared, total = _sequences(case)
            n = len(total)
            # the sequences of a group keep the whole chunks of their prefix once; the last, partly shared chunk is each one's copy
            own_chunks = [-(-t // CHUNK) - p // CHUNK for t, p in zip(total, [p for c, p in zip(counts, shared) for _ in range(c)])]
            pre = [p // CHUNK for p in shared]
            perm = torch.randperm(sum(pre) + sum(own_chunks), generator=gen)
            s["table"] = torch.zeros(n, max(-(-t // CHUNK) for t in total), dtype=torch.int64)
            s["pool"] = _pool(len(perm), q8, int(torch.randint(1 << 30, (1,), generator=gen)), True)
            at, i = 0, 0
            for c, p, k in zip(counts, shared, pre):
                head = perm[at:at + k]
                at += k
                for j in range(i, i + c):
                    s["table"][j, :k] = head
                    s["table"][j, k:k + own_chunks[j]] = perm[at:at + own_chunks[j]]
                    at += own_chunks[j]
                    if p % CHUNK:
                        s["pool"][s["table"][j, k], :, :, :p % CHUNK] = s["pool"][s["table"][i, k], :, :, :p % CHUNK]
                i += c
            offsets = [0]
            for c in counts:
                offsets.append(offsets[-1] + c)
            s["group_off"], s["shared_len"], s["seq_len"] = ints(offsets), ints(shared), ints(total)
            s["max_shared"] = max(shared)
            s["max_tail"] = max(t - p for t, p in zip(total, [p for c, p in zip(counts, shared) for _ in range(c)]))
        s["q"] = (1.5 * torch.randn(n, HEADS, DIM, device="cuda", generator=dev)).to(kind)
        s["gate"] = torch.randn(n, HEADS, DIM, device="cuda", generator=dev).to(kind)
    s["chunk_ptrs"] = _addresses(s["pool"], s["table"])
    s["table"] = s["table"].cuda()
    return s


# ---- one pass -----------------------------------------------------------------------------

def run(s):
    return {"append": _append, "prefill": _prefill, "shared": _shared}[s["case"]["op"]](s)


def _q8_values(blocks):
    """What q8_0 blocks [..., 8, 34] stand for, as [..., 256] f16."""
    return torch.mul(blocks[..., 2:].view(torch.int8), blocks[..., :2].view(torch.float16)).flatten(-2)


def _append(s):
    case, pool = s["case"], s["pool"]
    if own:
        from qwowl35_b200 import ops
        q, gate = ops.attn_append(s["qkv"], s["q_norm"], s["k_norm"], s["freq"], s["rotary"], s["sections"], s["tok_seq"],
                                  s["tok_pos"], s["chunk_ptrs"], 0, s["v_off"], eps=EPS, interleaved=case["interleaved"],
                                  dtype=s["kind"], kv_q8=case["q8"])
    else:
        n = s["qkv"].shape[0]
        full = s["qkv"][:, :2 * HEADS * DIM].view(n, HEADS, 2, DIM)
        kv = s["qkv"][:, 2 * HEADS * DIM:].view(n, 2, KV_HEADS, DIM)
        pair = torch.arange(PAIRS, device="cuda")
        axis = torch.zeros_like(pair)
        if case["axes"] == 3:
            a, b, c = s["sections"]
            if case["interleaved"]:
                axis = torch.where((pair % 3 == 1) & (pair < 3 * b), 1, torch.where((pair % 3 == 2) & (pair < 3 * c), 2, 0))
            else:
                axis = (pair >= a).long() + (pair >= a + b).long()
        angle = s["rotary"].t()[:, axis].double() * s["freq"].double()  # far positions need 64 bits
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

        def turned(x, weight):
            y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
            lo, hi = y[..., :PAIRS], y[..., PAIRS:2 * PAIRS]
            return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, y[..., 2 * PAIRS:]], -1)

        q = turned(full[:, :, 0], s["q_norm"]).to(s["kind"])
        gate = full[:, :, 1].to(s["kind"], copy=True)
        rows = torch.stack([turned(kv[:, 0], s["k_norm"]), kv[:, 1]], 1)  # [n, K or V, head, dim]
        chunk, at = s["table"][s["tok_seq"].long(), s["tok_pos"].long() // CHUNK], s["tok_pos"].long() % CHUNK
        if case["q8"]:
            x = rows.unflatten(-1, (DIM // 32, 32))
            d = x.abs().amax(-1, keepdim=True) / 127
            v = x * torch.where(d > 0, 1 / d, torch.zeros_like(d))
            code = torch.where(v < 0, -torch.floor(0.5 - v), torch.floor(0.5 + v)).clamp(-127, 127).to(torch.int8)
            pool[chunk, :, :, at] = torch.cat([d.to(torch.float16).view(torch.uint8), code.view(torch.uint8)], -1)
        else:
            pool[chunk, :, :, at] = rows.to(torch.float16)
    if case["q8"]:
        chunk, at = s["table"][s["tok_seq"].long(), s["tok_pos"].long() // CHUNK], s["tok_pos"].long() % CHUNK
        return {"q": q, "gate": gate, "rows": _q8_values(pool[chunk, :, :, at])}
    return {"q": q, "gate": gate, "cache": pool}


def _keys(s, longest):
    """K and V of every sequence, padded to whole chunks: [n, kv head, position, dim] in 32 bits."""
    count = -(-longest // CHUNK)
    part = s["pool"][s["table"][:, :count]]
    if s["case"]["q8"]:
        part = (part[..., 2:].view(torch.int8).float() * part[..., :2].view(torch.float16).float()).flatten(-2)
    else:
        part = part.float()
    part = part.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)  # [K or V, n, head, position, dim]
    return part[0], part[1]


def _attend(q, gate, k, v, length, window, sink):
    """q, gate [n, t, head, dim], length [n, t] positions each query sees (0: none); f32 [n, t, head * dim]."""
    n, t = length.shape
    x = q.float().view(n, t, KV_HEADS, GROUP, DIM).permute(0, 2, 3, 1, 4).reshape(n, KV_HEADS, GROUP * t, DIM)
    score = (x @ k.transpose(-1, -2)) * (1 / math.sqrt(DIM))
    at = torch.arange(k.shape[2], device="cuda")
    size = length[..., None]
    seen = at < size
    if window > 0:
        kept = size.clamp(max=sink)
        seen = seen & ((kept + window >= size) | (at < kept) | (at >= size - window))
    score = score.view(n, KV_HEADS, GROUP, t, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    o = (p.view(n, KV_HEADS, GROUP * t, -1) @ v).view(n, KV_HEADS, GROUP, t, DIM) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, t, HEADS, DIM)
    return (o / (1 + torch.exp(-gate.float()))).flatten(2)


def _prefill(s):
    case = s["case"]
    if own:
        from qwowl35_b200 import ops
        return ops.gqa_prefill(s["q"], s["gate"], s["run_off"], s["seq_len"], s["max_run"], s["max_len"], s["chunk_ptrs"], 0,
                               s["v_off"], window=case["window"], sink=case["sink"], kv_q8=case["q8"])
    k, v = _keys(s, s["max_len"])
    begin, end = s["run_off"][:-1].long(), s["run_off"][1:].long()
    t = torch.arange(s["max_run"], device="cuda")
    real = t < (end - begin)[:, None]
    token = torch.where(real, begin[:, None] + t, 0)
    length = torch.where(real, s["seq_len"].long()[:, None] - (end - begin)[:, None] + t + 1, 0)
    o = _attend(s["q"][token], s["gate"][token], k, v, length, case["window"], case["sink"])
    return o[real].to(s["kind"])


def _shared(s):
    case = s["case"]
    if own:
        from qwowl35_b200 import ops
        return ops.gqa_decode_shared(s["q"], s["gate"], s["seq_len"], s["group_off"], s["shared_len"], s["max_shared"],
                                     s["max_tail"], s["chunk_ptrs"], 0, s["v_off"], window=case["window"], sink=case["sink"],
                                     kv_q8=case["q8"])
    k, v = _keys(s, s["table"].shape[1] * CHUNK)
    o = _attend(s["q"][:, None], s["gate"][:, None], k, v, s["seq_len"].long()[:, None], case["window"], case["sink"])
    return o[:, 0].to(s["kind"])


# ---- the definitions in 64 bits --------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    length = s["seq_len"].tolist()
    q, gate = s["q"].double(), s["gate"].double()
    out = torch.empty_like(q)
    for i, total in enumerate(length):
        pages = s["pool"][s["table"][i, :-(-total // CHUNK)]]
        if case["q8"]:
            pages = (pages[..., 2:].view(torch.int8).double() * pages[..., :2].view(torch.float16).double()).flatten(-2)
        first, last = (s["run_off"][i:i + 2].tolist() if case["op"] == "prefill" else (i, i + 1))
        for head in range(KV_HEADS):
            k, v = (pages[:, j, head].reshape(-1, DIM)[:total].double() for j in (0, 1))
            for h in range(head * GROUP, (head + 1) * GROUP):
                for a in range(first, last, 2048):
                    b = min(last, a + 2048)
                    # the row that ends the run sees every position; the one before it sees one less
                    see = total - (last - torch.arange(a, b, device="cuda"))[:, None] + 1
                    j = torch.arange(total, device="cuda")
                    mask = j < see
                    if case["window"] > 0:
                        few = torch.clamp(see, max=case["sink"])
                        mask &= (few + case["window"] >= see) | (j < few) | (j >= see - case["window"])
                    z = torch.where(mask, q[a:b, h] @ k.t() / math.sqrt(DIM), -math.inf)
                    out[a:b, h] = torch.softmax(z, -1) @ v * torch.sigmoid(gate[a:b, h])
    return out.flatten(1)


def _exact_append(s):
    case, x = s["case"], s["qkv"].double()
    n = x.shape[0]
    axis = [0] * PAIRS
    if case["axes"] == 3 and case["interleaved"]:
        axis = [i % 3 if i % 3 and i < 3 * s["sections"][i % 3] else 0 for i in range(PAIRS)]
    elif case["axes"] == 3:
        axis = [a for a in range(3) for _ in range(s["sections"][a])]
    angle = torch.stack([s["rotary"][a].double() * s["freq"][i].double() for i, a in enumerate(axis)], 1)[:, None]

    def head(part, weight):
        y = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + EPS) * weight.double()
        z = torch.complex(y[..., :PAIRS], y[..., PAIRS:2 * PAIRS]) * torch.polar(torch.ones_like(angle), angle)
        y[..., :PAIRS], y[..., PAIRS:2 * PAIRS] = z.real, z.imag
        return y

    heads = x[:, :2 * HEADS * DIM].view(n, HEADS, 2 * DIM)
    q, gate = head(heads[..., :DIM].clone(), s["q_norm"]), heads[..., DIM:].clone()
    k, v = x[:, 2 * HEADS * DIM:].view(n, 2, KV_HEADS, DIM).unbind(1)
    if case["q8"]:
        return {"q": q, "gate": gate, "rows": None}  # codes: whole steps, no value between them
    cache = s["pool"].double()
    k = head(k.clone(), s["k_norm"])
    where = s["table"][s["tok_seq"].long(), s["tok_pos"].long() // CHUNK], s["tok_pos"].long() % CHUNK
    cache[where[0], 0, :, where[1]] = k
    cache[where[0], 1, :, where[1]] = v
    return {"q": q, "gate": gate, "cache": cache}
