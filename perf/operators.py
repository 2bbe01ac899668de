"""The operators of a server that decodes many requests of unequal length together, as cases that can be timed: the pages of a
step, rotation and storage of its keys and values in 8 bits, attention over the pages, and the choice of the next tokens.

The cache.  Requests share a pool of pages; a page holds `block` tokens of every kv head.  Keys and values are int8 codes with one f32
scale for each page and head: scale = (largest magnitude written to the page so far) / 127, value = code * scale, code = value / scale rounded to
the nearest whole number, ties to even.  A page whose scale grows is coded again: code * old / new, rounded the same way.  In
memory both are ordered the way the products read them: keys [page, head, dim / 16, token, 16], values [page, head, token / 16, dim, 16].

paged_plan: request r has `lengths[r]` tokens in the cache and brings `new_tokens[r]`.  Pages that the new tokens need are taken from the
top of the stack free_blocks[:free_count], request after request; token t of the step gets its position and its slot, page * block +
position % block (-1 behind the last one).

prepare_paged_attention: entries d and d + n_freqs of every head of query and key turn by position * freqs[d]; keys and values go to their slots.

paged_attention: row i of request r is position context - rows + i and attends the positions up to its own, the last `window` of them where
a window is given: softmax(scale * q . k) . v over the coded keys and values.

sample_rows: w = exp((logit - largest) / temperature); of the tokens in the order of their logits (the lower index first
among equals) the first n stay: at most top_k, the fewest that hold top_p of the weight of those, none under min_p of the largest
weight.  Token = the first at which the weight so far passes u times the weight of all n; with its log-probability."""
from __future__ import annotations

import math
import random

import torch

own = False

# geometries of this repository's configurations (the second one of width 3584): heads, kv heads, head size
MISTRAL = dict(heads=32, kv_heads=8, head_dim=128)
WIDE = dict(heads=28, kv_heads=4, head_dim=128)
QWEN = dict(heads=14, kv_heads=2, head_dim=64)
ROPE_THETA = 1.0e6


def listed():
    return [
        # the bookkeeping of one decode step of a full batch
        dict(name="plan_decode_64", kind="plan", requests=64, shortest=16, longest=4000, new=1, prompts=0, block=32, mix=1),
        # requests that arrive with their prompts beside others that decode
        dict(name="plan_mixed_200", kind="plan", requests=200, shortest=1, longest=4000, new=600, prompts=25, block=16, mix=2),
        # one token of each request: f32 as the quantized projections give it
        dict(name="prepare_decode_48", kind="prepare", requests=48, shortest=16, longest=4000, new=1, prompts=0, block=32, dtype="float32", mix=3, **MISTRAL),
        # ragged prompts, bf16
        dict(name="prepare_prompts_5", kind="prepare", requests=5, shortest=0, longest=2000, new=900, prompts=5, block=64, dtype="bfloat16", mix=4, **MISTRAL),
        # the smallest call: one request's token at the headline context
        dict(name="attend_1_2048", kind="attend", requests=1, shortest=2048, longest=2048, new=1, prompts=0, block=32, window=0, dtype="float32", mix=5, **MISTRAL),
        # seven query heads to a kv head, heads of 64, short and middling contexts
        dict(name="attend_16_hd64", kind="attend", requests=16, shortest=200, longest=2500, new=1, prompts=0, block=16, window=0, dtype="float32", mix=6, **QWEN),
        # a full batch of very unequal contexts
        dict(name="attend_64_ragged", kind="attend", requests=64, shortest=100, longest=8000, new=1, prompts=0, block=32, window=0, dtype="bfloat16", mix=7, **MISTRAL),
        # the headline prompt, nothing cached before it, f32
        dict(name="attend_prompt_2048", kind="attend", requests=1, shortest=0, longest=0, new=2048, prompts=1, block=64, window=0, dtype="float32", mix=8, **MISTRAL),
        # portions of prompts behind long contexts beside single tokens, sliding window, bf16
        dict(name="attend_portions_12", kind="attend", requests=12, shortest=500, longest=6000, new=700, prompts=4, block=64, window=4096, dtype="bfloat16", mix=9, **WIDE),
        # a single stream's next token
        dict(name="sample_1_32000", kind="sample", rows=1, vocab=32000, dtype="float32", mix=10),
        # a small batch, large vocabulary
        dict(name="sample_16_151936", kind="sample", rows=16, vocab=151936, dtype="bfloat16", mix=11),
        # a full batch, every request with settings of its own
        dict(name="sample_64_152064", kind="sample", rows=64, vocab=152064, dtype="float32", mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "prepare", "attend", "attend", "sample"])
    if kind == "sample":
        return dict(kind=kind, rows=_spread(rng, 1, 64), vocab=_spread(rng, 1000, 152064), dtype=rng.choice(["float32", "bfloat16"]), mix=rng.randrange(1 << 20))
    form = rng.choice([MISTRAL, WIDE, QWEN, dict(heads=16, kv_heads=16, head_dim=64), dict(heads=24, kv_heads=2, head_dim=128)])
    prompts = rng.random() < 0.5
    case = dict(kind=kind, shortest=rng.choice([0, 1, 100]), longest=_spread(rng, 100, 6000), block=rng.choice([16, 32, 64, 128]), mix=rng.randrange(1 << 20))
    if kind == "plan":
        case |= dict(requests=_spread(rng, 1, 256), prompts=0, new=1)
        case |= dict(prompts=rng.randint(1, max(1, min(25, case["requests"]))), new=_spread(rng, 2, 600)) if prompts else {}
        return case
    case |= dict(dtype=rng.choice(["float32", "bfloat16"]), requests=_spread(rng, 1, 64), prompts=0, new=1, **form)
    if prompts:
        case |= dict(requests=rng.randint(1, 8), new=_spread(rng, 2, 700))
        case |= dict(prompts=rng.randint(1, case["requests"]))
        case |= dict(longest=min(case["longest"], 4000))
    if kind == "attend":
        case |= dict(window=rng.choice([0, 0, 4096, _spread(rng, 16, 2000)]))
    return case


def _lengths(case):
    """Tokens in the cache and new tokens of every request: of the case, not of the seed.  The first `prompts` requests bring prompts."""
    rng = random.Random(case["mix"])
    lo, hi = case["shortest"], max(case["shortest"], case["longest"])
    cached = [int(lo + (hi - lo) * rng.random() ** 1.5) if lo < hi else lo for _ in range(case["requests"])]
    new = [1] * case["requests"]
    for r in range(case["prompts"]):
        new[r] = case["new"] if case["prompts"] == 1 else rng.randint(max(1, case["new"] // 8), case["new"])
    if case["kind"] == "plan" and case["requests"] > 4:
        new[-2] = 0  # one request waits
    return cached, new


def _visible(case):
    """Query rows' attended positions in all, and cached positions that some row attends."""
    cached, new = _lengths(case)
    pairs = rows = 0
    for c, n in zip(cached, new):
        w = case["window"] or c + n
        pairs += sum(min(w, c + i + 1) for i in range(n))
        rows += min(c + n, w + n - 1)
    return pairs, rows


def work(case):
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 40), "flops": case["rows"] * case["vocab"] * 4}
    cached, new = _lengths(case)
    tokens, block = sum(new), case["block"]
    if case["kind"] == "plan":
        pages = sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(cached, new))
        return {"bytes": 20 * case["requests"] + 8 * tokens + 8 * pages, "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2
    q, kv = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    if case["kind"] == "prepare":
        shown = sum(c % block + n for c, n in zip(cached, new))  # rows of the pages written to, read back in f32
        return {"bytes": tokens * (2 * q + 2 * kv) * size + 2 * kv * (tokens + sum(c % block for c in cached)) + 2 * kv * shown * 5, "flops": tokens * (3 * (q + kv) + 4 * kv)}
    pairs, rows = _visible(case)
    return {"bytes": 2 * kv * rows + 8 * case["kv_heads"] * rows // block + 2 * tokens * q * size, "flops": 4 * pairs * q}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + case["mix"])

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # some rows nearly decided, some with thousands of likely tokens
        logits = (randn(rows, vocab) * (1.0 + 3.0 * rand(rows, 1))).to(getattr(torch, case["dtype"]))
        pick = torch.randint(0, 4, (4, rows), generator=gen, device="cuda")
        temperature = 0.5 + 0.8 * rand(rows)
        top_k = torch.tensor([0, 20, 50, 400], dtype=torch.int32, device="cuda")[pick[0]]
        top_p = torch.tensor([1.0, 0.8, 0.9, 0.98], device="cuda")[pick[1]]
        min_p = torch.tensor([0.0, 0.0, 0.02, 0.1], device="cuda")[pick[2]]
        u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
        return dict(case=case, logits=logits, u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, tokens=torch.empty(rows, dtype=torch.int32, device="cuda"),
                    logprobs=torch.empty(rows, device="cuda"))

    cached, new = _lengths(case)
    block, requests, tokens = case["block"], case["requests"], sum(new)
    blocks = [-(-(c + n) // block) for c, n in zip(cached, new)]
    width = max(blocks) + 2
    pages = sum(blocks) + 8
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = dict(case=case, block=block)
    if case["kind"] == "plan":
        held = [-(-c // block) for c in cached]
        table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for r, h in enumerate(held):
            table[r, :h] = order[at:at + h]
            at += h
        free = torch.zeros(pages, dtype=torch.int32, device="cuda")
        free[:pages - at] = order[at:]
        capacity = tokens + tokens // 16 + 3  # room for padding, as a captured step has it
        return s | dict(lengths=ints(cached), new_tokens=ints(new), table=table, free=free, free_count=ints([pages - at]), capacity=capacity, context=ints([0] * requests),
                        query_start=ints([0] * (requests + 1)), positions=ints([0] * capacity), slots=ints([0] * capacity), left=ints([0]), status=ints([0]))
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    dtype = getattr(torch, case["dtype"])
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(blocks):
        table[r, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s |= dict(table=table, query_start=ints(starts), context=ints([c + n for c, n in zip(cached, new)]), max_query=max(new), max_context=max(c + n for c, n in zip(cached, new)))
    # what the cache holds: codes of roughly normal entries whose largest is 127, scales that differ by page and head
    s["k_codes"] = (randn(pages, kv, hd // 16, block, 16) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["v_codes"] = (randn(pages, kv, block // 16, hd, 16) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["k_scales"] = (0.5 + rand(pages, kv)) * (3.5 / 127)
    s["v_scales"] = (0.5 + rand(pages, kv)) * (3.5 / 127)
    s["query"] = randn(tokens, heads, hd).to(dtype)
    if own:  # what a server makes once: the handle of its cache, the workspace of its attention
        from kmll_b200 import ops
        s["cache"] = ops.DevicePagedI8Cache.from_parts(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
    if case["kind"] == "attend":
        s |= dict(out=torch.zeros(tokens, heads * hd, dtype=dtype, device="cuda"), scale=1.0 / math.sqrt(hd))
        if own:
            s["workspace"] = ops.paged_attention_workspace(s["cache"], heads, requests, tokens, s["max_query"], s["max_context"])
        return s
    s["key"], s["value"] = randn(tokens, kv, hd).to(dtype), randn(tokens, kv, hd).to(dtype)
    s["freqs"] = torch.tensor([ROPE_THETA ** (-2.0 * d / hd) for d in range(hd // 2)], dtype=torch.float32, device="cuda")
    positions = [c + i for c, n in zip(cached, new) for i in range(n)]
    owner = ints([r for r, n in enumerate(new) for _ in range(n)]).long()
    s["positions"] = ints(positions)
    at = s["positions"].long()
    s["slots"] = (table[owner, at // block] * block + at % block).to(torch.int32)
    # every row of the pages that the step writes to
    shown = [(r, i) for r, (c, n) in enumerate(zip(cached, new)) for i in range(c - c % block, c + n)]
    owner, at = ints([r for r, _ in shown]).long(), ints([i for _, i in shown]).long()
    s["shown"] = (table[owner, at // block] * block + at % block).to(torch.int32)
    s["turned"] = torch.empty_like(s["query"])
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _plan(s):
    block, lengths, new, table, cap = s["block"], s["lengths"].long(), s["new_tokens"].long(), s["table"], s["capacity"]
    requests, width = table.shape
    held, wanted = -(-lengths // block), -(-(lengths + new) // block)
    end, taken = torch.cumsum(new, 0), torch.cumsum(wanted - held, 0)
    count = s["free_count"].long()
    fine = (taken[-1:] <= count) & (wanted.max() <= width) & (end[-1:] <= cap) & (new.min() >= 0) & (lengths.min() >= 0)
    t = torch.arange(cap, device="cuda")
    r = torch.searchsorted(end, t, right=True).clamp_(max=requests - 1)
    valid = (t < end[-1]) & fine
    pos = torch.where(valid, lengths[r] + t - (end - new)[r], 0)
    at = torch.where(valid, pos // block, 0)
    fresh = valid & (at >= held[r])
    place = count - 1 - ((taken - wanted + held)[r] + at - held[r])
    page = torch.where(fresh, s["free"][place.clamp(0, s["free"].numel() - 1)].long(), table[r, at].long())
    padded = torch.cat([table, table[:, :1]], 1)
    padded[r, torch.where(fresh, at, width)] = page.to(torch.int32)
    table.copy_(padded[:, :width])
    start = torch.cat([torch.zeros_like(end[:1]), end]) * fine
    return dict(context=torch.where(fine, lengths + new, lengths).to(torch.int32), query_start=start.to(torch.int32), table=table, positions=pos.to(torch.int32),
                slots=torch.where(valid, page * block + pos % block, -1).to(torch.int32), left=torch.where(fine, count - taken[-1:], count).to(torch.int32),
                status=(~fine).to(torch.int32))


def _turned(x, positions, freqs):
    """64 bits: positions are far from 0, and the codes of the keys must not depend on how an angle is rounded."""
    half = freqs.numel()
    angle = positions.double()[:, None, None] * freqs.double()
    c, n = angle.cos(), angle.sin()
    a, b = x[..., :half].double(), x[..., half:2 * half].double()
    return torch.cat([a * c - b * n, a * n + b * c, x[..., 2 * half:].double()], -1)


def _store(x, slots, block, rows, scales):
    """x [tokens, heads, dim] (64 bits) into rows [page, token, head, dim] of codes with scales [page, head]: all of both, updated."""
    pages = rows.shape[0]
    page, at = slots.long() // block, slots.long() % block
    largest = torch.zeros(pages, x.shape[1], dtype=torch.float64, device=x.device).index_reduce_(0, page, x.abs().amax(-1), "amax")
    fresh = torch.zeros(pages, dtype=torch.int64, device=x.device).index_reduce_(0, page, (at == 0).long(), "amax") > 0
    before = torch.where(fresh[:, None], 0.0, scales)
    scale = torch.maximum(before, (largest / 127.0).float())
    grown = (scale > scales) | fresh[:, None]
    divisor = torch.where(scale > 0, scale, 1.0).double()
    again = (rows.double() * before.double()[:, None, :, None] / divisor[:, None, :, None]).round()
    rows = torch.where(grown[:, None, :, None], again, rows.double())
    scale = torch.where(grown, scale, scales)
    rows[page, at] = (x / divisor[page][..., None]).round().clamp(-127, 127)
    return rows, scale


def _prepare(s):
    case, block = s["case"], s["block"]
    kv, hd = case["kv_heads"], case["head_dim"]
    pages = s["k_codes"].shape[0]
    turned = _turned(s["query"], s["positions"], s["freqs"]).to(s["query"].dtype)
    key = _turned(s["key"], s["positions"], s["freqs"])
    # only the pages of this step take part
    page, back = torch.unique(s["shown"].long() // block, return_inverse=True)
    place = torch.zeros(pages, dtype=torch.int64, device="cuda")
    place[page] = torch.arange(page.numel(), device="cuda")
    slots = place[s["slots"].long() // block] * block + s["slots"].long() % block
    k, ks = _store(key, slots, block, s["k_codes"][page].permute(0, 3, 1, 2, 4).reshape(-1, block, kv, hd), s["k_scales"][page])
    v, vs = _store(s["value"].double(), slots, block, s["v_codes"][page].permute(0, 2, 4, 1, 3).reshape(-1, block, kv, hd), s["v_scales"][page])
    s["k_codes"][page] = k.to(torch.int8).view(-1, block, kv, hd // 16, 16).permute(0, 2, 3, 1, 4)
    s["v_codes"][page] = v.to(torch.int8).view(-1, block // 16, 16, kv, hd).permute(0, 3, 1, 4, 2)
    s["k_scales"][page], s["v_scales"][page] = ks, vs
    at = s["shown"].long() % block
    return dict(query=turned, key=k[back, at].float() * ks[back][..., None], value=v[back, at].float() * vs[back][..., None])


def _attend(s):
    case, block, context, start = s["case"], s["block"], s["context"].long(), s["query_start"].long()
    heads, kv, hd, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    tokens, requests, most = s["query"].shape[0], context.numel(), -(-s["max_context"] // block)
    pages = s["table"][:, :most].long().clamp(min=0)
    k = (s["k_codes"][pages].float() * s["k_scales"][pages][..., None, None, None]).permute(0, 2, 1, 4, 3, 5).reshape(requests, kv, most * block, hd)
    v = (s["v_codes"][pages].float() * s["v_scales"][pages][..., None, None, None]).permute(0, 2, 1, 3, 5, 4).reshape(requests, kv, most * block, hd)
    rows = start[1:] - start[:-1]
    i = torch.arange(s["max_query"], device="cuda")
    there = i < rows[:, None]
    row = torch.where(there, start[:-1, None] + i, 0)
    q = s["query"].float()[row].view(requests, -1, kv, heads // kv, hd).permute(0, 2, 3, 1, 4) * s["scale"]
    scores = torch.matmul(q.reshape(requests, kv, -1, hd), k.transpose(2, 3)).view(requests, kv, heads // kv, -1, most * block)
    pos = (context - rows)[:, None] + i
    j = torch.arange(most * block, device="cuda")
    seen = (j <= pos[..., None]) & there[..., None]
    if window:
        seen &= j > pos[..., None] - window
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e38))
    y = torch.matmul(weights.view(requests, kv, -1, most * block), v).view(requests, kv, heads // kv, -1, hd)
    y = y / weights.sum(-1, keepdim=True).clamp(min=1e-38)
    out = torch.cat([s["out"], s["out"][:1]])
    out[torch.where(there, row, tokens)] = y.permute(0, 3, 1, 2, 4).reshape(requests, -1, heads * hd).to(out.dtype)
    return s["out"].copy_(out[:tokens])


def _sample(s):
    """64 bits: a sum that ends a unit beside u times the whole would choose another token."""
    x, order = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
    vocab = x.shape[1]
    w = torch.exp((x - x[:, :1]) / s["temperature"].double()[:, None])
    sums = torch.cumsum(w, 1)
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab).clamp(max=vocab).long()[:, None]
    share = s["top_p"].double()[:, None] * sums.gather(1, k - 1)
    n = torch.minimum(k, torch.where(s["top_p"][:, None] < 1, torch.searchsorted(sums, share) + 1, vocab))
    n = torch.minimum(n, (w >= s["min_p"].double()[:, None]).sum(1, keepdim=True)).clamp_(min=1)
    whole = sums.gather(1, n - 1)
    at = torch.minimum(torch.searchsorted(sums, s["u"][:, None] * whole, right=True), n - 1)
    return dict(tokens=order.gather(1, at)[:, 0].to(torch.int32), logprobs=(w.gather(1, at) / whole).log()[:, 0].float())


PLAIN = dict(plan=_plan, prepare=_prepare, attend=_attend, sample=_sample)


def run(s):
    if not own:
        return PLAIN[s["case"]["kind"]](s)
    from kmll_b200 import ops
    kind = s["case"]["kind"]
    if kind == "plan":
        ops.paged_plan(s["lengths"], s["new_tokens"], s["block"], s["table"], s["free"], s["free_count"], s["context"], s["query_start"], s["positions"], s["slots"], s["left"],
                       s["status"])
        return {k: s[k] for k in ("context", "query_start", "table", "positions", "slots", "left", "status")}
    if kind == "prepare":
        turned = ops.prepare_paged_attention(s["query"], s["key"], s["value"], s["freqs"], s["positions"], s["slots"], s["cache"], query_rot=s["turned"])
        k, v = ops.paged_cache_rows(s["cache"], s["shown"])
        return dict(query=turned, key=k, value=v)
    if kind == "attend":
        return ops.paged_attention(s["query"], s["query_start"], s["context"], s["table"], s["cache"], s["max_query"], s["max_context"], s["scale"], s["case"]["window"],
                                   workspace=s["workspace"], out=s["out"])
    tokens, logprobs = ops.sample_rows(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], tokens=s["tokens"], logprobs=s["logprobs"])
    return dict(tokens=tokens, logprobs=logprobs)


# ---- 64 bits, request by request --------------------------------------------------------------------------------------------
def _exact_plan(s):
    block, table = s["block"], s["table"].cpu().clone()
    lengths, new, free, count = s["lengths"].tolist(), s["new_tokens"].tolist(), s["free"].tolist(), s["free_count"].item()
    start, positions, slots = [0], [], []
    for r, (c, n) in enumerate(zip(lengths, new)):
        for pos in range(c, c + n):
            if pos % block == 0:
                count -= 1
                table[r, pos // block] = free[count]
            positions.append(pos)
            slots.append(int(table[r, pos // block]) * block + pos % block)
        start.append(len(positions))
    more = s["capacity"] - len(positions)
    as_ints = {k: torch.tensor(v, dtype=torch.int32) for k, v in dict(context=[c + n for c, n in zip(lengths, new)], query_start=start, positions=positions + [0] * more,
                                                                      slots=slots + [-1] * more, left=[count], status=[0]).items()}
    return as_ints | dict(table=table)


def _exact_prepare(s):
    case, block = s["case"], s["block"]
    half = s["freqs"].numel()
    angle = torch.outer(s["positions"].double(), s["freqs"].double())[:, None, :]

    def turn(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.polar(torch.ones_like(angle), angle)
        return torch.cat([z.real, z.imag], -1)

    slots, shown = s["slots"].tolist(), s["shown"].tolist()
    mine = {}  # page -> (tokens of the step, their places)
    for t, slot in enumerate(slots):
        mine.setdefault(slot // block, ([], []))[0].append(t)
        mine[slot // block][1].append(slot % block)

    def stored(x, codes, scales):
        held = {}
        for page, (t, at) in mine.items():
            rows, old = codes[page], scales[page].double()  # [head, token, dim], [head]
            if 0 in at:
                rows, old = torch.zeros_like(rows), torch.zeros_like(old)
            scale = torch.maximum(old, (x[t].abs().amax((0, 2)) / 127).float().double())
            factor = torch.where(scale > old, old / scale, torch.ones_like(old))
            rows = torch.round(rows.double() * factor[:, None, None])
            rows[:, at] = torch.round(x[t] / scale[None, :, None]).permute(1, 0, 2)
            held[page] = rows * scale[:, None, None]
        return torch.stack([held[i // block][:, i % block] for i in shown])

    k_rows = s["k_codes"].permute(0, 1, 3, 2, 4).flatten(3)
    v_rows = s["v_codes"].permute(0, 1, 2, 4, 3).flatten(2, 3)
    return dict(query=turn(s["query"]), key=stored(turn(s["key"]), k_rows, s["k_scales"]), value=stored(s["value"].double(), v_rows, s["v_scales"]))


def _exact_attend(s):
    case, block, hd = s["case"], s["block"], s["case"]["head_dim"]
    group = case["heads"] // case["kv_heads"]
    out = s["out"].double()
    start, context = s["query_start"].tolist(), s["context"].tolist()
    for r, c in enumerate(context):
        a, b = start[r], start[r + 1]
        if a == b:
            continue
        pages = s["table"][r, :-(-c // block)].long()
        k = (s["k_codes"][pages].permute(1, 0, 3, 2, 4).flatten(3).double() * s["k_scales"][pages].t()[:, :, None, None].double()).flatten(1, 2)[:, :c]
        v = (s["v_codes"][pages].permute(1, 0, 2, 4, 3).flatten(2, 3).double() * s["v_scales"][pages].t()[:, :, None, None].double()).flatten(1, 2)[:, :c]
        j = torch.arange(c, device="cuda")
        for g in range(group):
            q = s["query"][a:b, g::group].transpose(0, 1).double()
            z = torch.bmm(q, k.transpose(1, 2)) * s["scale"]
            pos = torch.arange(c - (b - a), c, device="cuda")[:, None]
            hidden = (j > pos) | (j <= pos - case["window"]) if case["window"] else j > pos
            y = torch.bmm(torch.softmax(z.masked_fill(hidden, -math.inf), -1), v)
            out.view(out.shape[0], case["kv_heads"], group, hd)[a:b, :, g] = y.transpose(0, 1)
    return out


def _exact_sample(s):
    tokens, logprobs = [], []
    for row, u, temperature, k, p, least in zip(s["logits"].double().cpu(), s["u"].tolist(), s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist()):
        order = sorted(range(row.numel()), key=row.neg().tolist().__getitem__)
        w = torch.exp((row[order] - row.max()) / temperature)
        w = w[:k] if k else w
        sums = w.cumsum(0)
        if p < 1:
            w = w[:int((sums < p * sums[-1]).sum()) + 1]
        w = w[w >= least]
        sums = w.cumsum(0)
        at = min(int((sums <= u * sums[-1]).sum()), w.numel() - 1)
        tokens.append(order[at])
        logprobs.append(math.log(w[at] / sums[-1]))
    return dict(tokens=torch.tensor(tokens, dtype=torch.int32), logprobs=torch.tensor(logprobs, dtype=torch.float64))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample" and case["rows"] * case["vocab"] > 12_000_000:
        return None
    return dict(plan=_exact_plan, prepare=_exact_prepare, attend=_exact_attend, sample=_exact_sample)[case["kind"]](s)
