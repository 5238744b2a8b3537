"""The operators that serve many requests at once, as measurable cases.

Kinds:
  plan       the pages, slots and positions of one step's new tokens, from the requests' lengths
             (lm_page_plan)
  attention  multi-head latent attention of every request's new tokens over the pages of a shared
             latent cache, queries absorbed into the latent space (lm_paged_attention)
  sample     the next tokens of a batch of logit rows, from temperature, top-k, top-p, min-p and
             given random numbers (lm_sample)

Sizes are DeepSeek-V2's and V2-Lite's: latent 512 and 64 rotary channels, 16 or 128 heads, pages of
16 to 128 tokens, a vocabulary of 102400 (and other ones).
"""
import math
import random

import numpy as np
import torch

own = False  # False: elementary torch operations; True: litemind_amd's operators

RANK, ROPE = 512, 64
WIDTH = RANK + ROPE
SCALE = (0.1 * 0.707 * math.log(40.0) + 1.0) ** 2 / math.sqrt(192.0)  # DeepSeek-V2-Lite's softmax scale
VOCAB = 102400
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ----

def _plan(requests, new, context, page, over, mix):
    return {"op": "plan", "requests": requests, "new": new, "context": context, "page": page, "over": over, "mix": mix}


def _attention(requests, chunks, new, context, heads=16, page=64, dtype="fp16", mix=0):
    return {"op": "attention", "requests": requests, "chunks": chunks, "new": new, "context": context, "heads": heads,
            "page": page, "dtype": dtype, "mix": mix}


def _sample(rows, vocab, filters, grid):
    return {"op": "sample", "rows": rows, "vocab": vocab, "filters": filters, "grid": grid}


def listed():
    def named(name, case):
        return {"name": name, **case}

    return [
        # a decode step of 48 conversations, two of which ended: the call before every step
        named("plan_decode_48", _plan(48, 1, 4000, 64, 2, 1)),
        # 509 requests, a part of them with prompt chunks: the step with the most tokens
        named("plan_chunks_509", _plan(509, 64, 3001, 16, 9, 2)),
        # one token of one conversation of ordinary length: the smallest call, latency counts
        named("attention_decode_1", _attention(1, 0, 1, 4000)),
        # one token of 32 conversations of uneven length
        named("attention_decode_32", _attention(32, 0, 1, 3999, mix=3)),
        # the larger model's 128 heads, 16 conversations
        named("attention_decode_heads_128", _attention(16, 0, 1, 2500, heads=128, mix=4)),
        # one token after a very long document, pages of 128
        named("attention_decode_long", _attention(1, 0, 1, 131071, page=128)),
        # a chunk of a prompt after the chunks before it
        named("attention_chunk_512", _attention(1, 1, 512, 3001)),
        # a step that mixes three prompt chunks with 21 decoding conversations, small pages, bf16
        named("attention_mixed_24", _attention(24, 3, 301, 2047, page=16, dtype="bf16", mix=5)),
        # whole prompts into empty pages
        named("attention_prompt_2048", _attention(1, 1, 2048, 0)),
        # the next token of one conversation
        named("sample_1", _sample(1, VOCAB, "mixed", False)),
        # the next tokens of a batch, logits on a bf16 grid (many ties), every row its own settings
        named("sample_32", _sample(32, VOCAB, "mixed", True)),
        # a large batch with temperature alone: nothing is cut off
        named("sample_256", _sample(256, VOCAB, "temperature", False)),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "attention", "attention", "attention", "attention", "sample", "sample"])
    mix = rng.randrange(1, 1 << 30)
    if op == "plan":
        requests = _log_uniform(rng, 1, 500)
        new = _log_uniform(rng, 1, max(1, min(2048, 16000 // requests)))
        return _plan(requests, new, _log_uniform(rng, 1, 4000), rng.choice([16, 32, 64, 128]),
                     rng.randrange(0, requests // 4 + 1), mix)
    if op == "sample":
        vocab = rng.choice([VOCAB, VOCAB, _log_uniform(rng, 300, 160000)])
        return _sample(_log_uniform(rng, 1, min(256, 256 * VOCAB // vocab)), vocab,
                       rng.choice(["temperature", "top_k", "top_p", "min_p", "mixed", "mixed"]), rng.random() < 0.5)
    page, dtype = rng.choice([16, 32, 64, 64, 128]), rng.choice(["fp16", "fp16", "bf16"])
    heads = rng.choice([16, 16, 16, 128, rng.choice([1, 4, 8, 20, 40, 64])])
    use = rng.choice(["decode", "decode", "long", "chunk", "prompt", "mixed"])
    if use == "decode":
        requests = _log_uniform(rng, 1, 48 if heads <= 64 else 16)
        return _attention(requests, 0, 1, _log_uniform(rng, 16, 4096), heads, page, dtype, mix)
    if use == "long":
        return _attention(1, 0, 1, _log_uniform(rng, 8192, 131071), min(heads, 16), page, dtype, mix)
    if use == "mixed":
        requests = _log_uniform(rng, 2, 24)
        return _attention(requests, rng.randrange(1, min(requests, 4)), _log_uniform(rng, 2, 300),
                          _log_uniform(rng, 16, 2047), min(heads, 16), page, dtype, mix)
    heads = min(heads, 64)
    new = _log_uniform(rng, 2, 2048 * 16 // max(16, heads))
    context = 0 if use == "prompt" else _log_uniform(rng, 1, max(1, min(4000, (1 << 21) * 16 // (max(16, heads) * new) - new)))
    return _attention(1, 1, new, context, heads, page, dtype, mix)


# ---- inputs, from the seed alone ----

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(case):
    """Cached and new tokens of every request: uneven, the first at the case's own sizes."""
    rng, R = random.Random(case["mix"]), case["requests"]
    if case["op"] == "plan":
        cached = [case["context"]] + [rng.randint(0, case["context"]) for _ in range(R - 1)]
        added = [case["new"]] + [rng.choice([1, rng.randint(0, case["new"])]) for _ in range(R - 1)]
        for r in rng.sample(range(R), case["over"]):
            added[r] = -1
        return cached, added
    low = case["context"] // 8
    cached = [case["context"]] + [rng.randint(low, case["context"]) for _ in range(R - 1)]
    added = [case["new"]] + [rng.randint(1, case["new"]) if r < case["chunks"] else 1 for r in range(1, R)]
    return cached, added


def _table(g, held, page, width, pages):
    """Block tables of requests that hold `held` tokens, their pages scattered over the pool as long service leaves
    them, and the pages that nobody holds."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    counts = torch.tensor([_pages(h, page) for h in held], device="cuda")
    column = torch.arange(width, device="cuda")
    taken = column[None] < counts[:, None]
    at = (counts.cumsum(0) - counts)[:, None] + column[None]
    table = torch.where(taken, order[at.clamp(max=pages - 1)], -1).to(torch.int32)
    return table.contiguous(), order[int(counts.sum()):].contiguous()


def _inputs(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.2
        # a few words stand out, as the context makes them
        likely = torch.randint(0, vocab, (rows, 40), generator=g, device="cuda")
        raised = torch.randn((rows, 40), generator=g, device="cuda").abs() * 4.0
        logits.scatter_add_(1, likely, raised)
        if case["grid"]:
            logits = logits.bfloat16().float()
        u = torch.rand((rows,), generator=g, device="cuda")

        def pick(values, where):
            if case["filters"] not in (where, "mixed"):
                return None
            at = torch.randint(0, len(values), (rows,), generator=g, device="cuda")
            return torch.tensor(values, device="cuda")[at]

        temperature = 0.5 + torch.rand((rows,), generator=g, device="cuda")
        if case["filters"] == "mixed":
            temperature[torch.rand((rows,), generator=g, device="cuda") < 0.05] = 0.0  # greedy rows
        params = torch.zeros((rows, 4), device="cuda")
        params[:, 0] = temperature
        params[:, 2] = 1.0
        top_k, top_p, min_p = (pick([0, 1, 20, 50, 400], "top_k"), pick([1.0, 0.95, 0.9, 0.5], "top_p"),
                               pick([0.0, 0.02, 0.1], "min_p"))
        if top_k is not None:
            params[:, 1] = top_k.to(torch.int32).view(torch.float32)  # whole numbers in their own bits
        if top_p is not None:
            params[:, 2] = top_p
        if min_p is not None:
            params[:, 3] = min_p
        return {"logits": logits.contiguous(), "params": params, "u": u}
    cached, added = _lengths(case)
    page = case["page"]
    total = [0 if a < 0 else c + a for c, a in zip(cached, added)]
    width = max(_pages(max(c, t), page) for c, t in zip(cached, total)) + 1
    if op == "plan":
        pages = sum(_pages(max(c, t), page) for c, t in zip(cached, total)) + 37
        table, free = _table(g, cached, page, width, pages)
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        head = pages - free.numel() // 2  # the free pages go round the ring's end
        ring[(head + torch.arange(free.numel(), device="cuda")) % pages] = free
        return {"cached": _ints(cached), "added": _ints(added), "table": table, "ring": ring,
                "queue": _ints([head % pages, free.numel()]), "pages": pages, "width": width,
                "tokens": sum(max(a, 0) for a in added) + 3}
    pages = sum(_pages(t, page) for t in total) + 5
    table, _ = _table(g, total, page, width, pages)
    dtype, tokens = DTYPES[case["dtype"]], sum(added)
    pool = torch.randn((pages, page, WIDTH), generator=g, device="cuda", dtype=dtype)
    pool[..., RANK:] *= 0.9
    q = torch.randn((tokens, case["heads"], WIDTH), generator=g, device="cuda") * 0.7
    starts = [0]
    for a in added:
        starts.append(starts[-1] + a)
    return {"cached": _ints(cached), "lengths": _ints(total), "starts": _ints(starts), "table": table.clamp(min=0),
            "pool": pool, "q": q.to(dtype), "pages": pages, "width": width, "tokens": tokens,
            "most_keys": max(total), "most_new": max(added)}


# ---- what a program holds before the call ----

class State:
    """The call's inputs, and with `own` a context and the buffers that it writes."""

    def __init__(self, case, seed):
        self.case, self.p, self.ctx = case, _inputs(case, seed), None
        if not own:
            return
        import litemind_amd as lm
        from litemind_amd import workload as wl

        self.ctx, p, op = lm.Context(wl.V2_LITE.moe_config(num_layers=1)), self.p, case["op"]

        def buffer(*shape, dtype=torch.int32):
            return torch.zeros(shape, device="cuda", dtype=dtype)

        if op == "sample":
            self.token, self.probability = buffer(case["rows"]), buffer(case["rows"], dtype=torch.float32)
        else:
            R, T = case["requests"], p["tokens"]
            self.step = step = lm.PagedStep(requests=R, tokens=T, pages=p["pages"], page_size=case["page"],
                                            table_width=p["width"])
            step.table = p["table"].data_ptr()
            if op == "plan":
                self.out = out = {"lengths": buffer(R), "starts": buffer(R + 1), "positions": buffer(T),
                                  "slots": buffer(T), "queue": buffer(2), "info": buffer(4)}
                step.max_added = max(case["new"], 1)
                step.cached, step.added = p["cached"].data_ptr(), p["added"].data_ptr()
                step.ring, step.queue_in = p["ring"].data_ptr(), p["queue"].data_ptr()
                step.queue_out, step.lengths = out["queue"].data_ptr(), out["lengths"].data_ptr()
                step.starts, step.positions = out["starts"].data_ptr(), out["positions"].data_ptr()
                step.slots, step.info = out["slots"].data_ptr(), out["info"].data_ptr()
            else:
                step.max_added = p["most_new"]
                step.lengths, step.starts = p["lengths"].data_ptr(), p["starts"].data_ptr()
                self.dtype = lm.DT_F16 if case["dtype"] == "fp16" else lm.DT_BF16
                self.y = buffer(T, case["heads"], RANK, dtype=DTYPES[case["dtype"]])
        torch.cuda.synchronize()

    def __del__(self):
        if getattr(self, "ctx", None) is not None and self.ctx.handle:
            self.ctx.synchronize()
            self.ctx.close()


def prepare(case, seed):
    return State(case, seed)


# ---- one pass ----

def run(s):
    op, p = s.case["op"], s.p
    if not own:
        return _plain_plan(s.case, p) if op == "plan" else _plain_attention(s.case, p) if op == "attention" \
            else _plain_sample(p)
    if op == "plan":
        s.ctx.page_plan(s.step)
        return {**s.out, "table": p["table"], "ring": p["ring"]}
    if op == "attention":
        s.ctx.paged_attention(s.step, p["q"].data_ptr(), p["pool"].data_ptr(), s.case["heads"], SCALE, s.y.data_ptr(),
                              dtype=s.dtype)
        return {"y": s.y}
    s.ctx.sample(p["logits"].data_ptr(), s.case["rows"], s.case["vocab"], p["params"].data_ptr(), p["u"].data_ptr(),
                 s.token.data_ptr(), probability=s.probability.data_ptr())
    return {"token": s.token, "probability": s.probability}


def _plain_plan(case, p):
    page, pages, T = case["page"], p["pages"], p["tokens"]
    cached, added, table, ring = p["cached"].long(), p["added"].long(), p["table"].long(), p["ring"].long()
    head, free = p["queue"][0].long(), p["queue"][1].long()
    over = added < 0
    new = added.clamp(min=0)
    lengths = torch.where(over, 0, cached + new)
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    had = (cached + page - 1) // page
    grown = torch.where(over, 0, (lengths + page - 1) // page - had)
    first = grown.cumsum(0) - grown
    column = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (column >= had[:, None]) & (column < (had + grown)[:, None])
    table = torch.where(fresh, ring[(head + first[:, None] + column - had[:, None]) % pages], table)
    # over requests' pages, in request and column order, behind the ring's last free page
    back = over[:, None] & (column < had[:, None])
    place = (back.reshape(-1).cumsum(0) - 1).view(back.shape)
    spot = torch.where(back, (head + free + place) % pages, pages)
    ring = torch.cat([ring, ring[:1]]).scatter(0, spot.reshape(-1), table.reshape(-1))[:pages]
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=new.numel() - 1)
    used = t < starts[-1]
    position = torch.where(used, cached[r] + t - starts[r], 0)
    slot = torch.where(used, table[r, position // page] * page + position % page, -1)
    taken, released = grown.sum(), back.sum()
    queue = torch.stack([(head + taken) % pages, free - taken + released])
    info = torch.stack([torch.zeros_like(taken), starts[-1], taken, released])
    whole = {"lengths": lengths, "starts": starts, "positions": position, "slots": slot, "queue": queue, "info": info,
             "table": table, "ring": ring}
    return {k: v.to(torch.int32) for k, v in whole.items()}


def _plain_attention(case, p):
    heads, page, R = case["heads"], case["page"], case["requests"]
    K, Q, T = p["most_keys"], p["most_new"], p["tokens"]
    starts, lengths = p["starts"].long(), p["lengths"].long()
    cached = lengths - (starts[1:] - starts[:-1])
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    i = t - starts[r]
    j = torch.arange(K, device="cuda")
    slot = p["table"].long()[:, j // page] * page + j % page
    keys = p["pool"].view(-1, WIDTH)[slot].float()                      # [R, K, 576]
    q = torch.zeros((R, Q, heads, WIDTH), device="cuda")
    q[r, i] = p["q"].float()
    s = (q.view(R, Q * heads, WIDTH) @ keys.transpose(1, 2).contiguous()).mul_(SCALE).view(R, Q, heads, K)
    last = cached[:, None] + torch.arange(Q, device="cuda")[None]
    s.masked_fill_((j[None, None] > last[..., None])[:, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1)
    y = (s.view(R, Q * heads, K) @ keys[..., :RANK].contiguous()).view(R, Q, heads, RANK) / total[..., None]
    return {"y": y[r, i].to(p["q"].dtype)}


def _plain_sample(p):
    logits, params, u = p["logits"].double(), p["params"], p["u"].double()
    temperature, top_p, min_p = params[:, 0].double(), params[:, 2].double(), params[:, 3].double()
    top_k = params[:, 1].contiguous().view(torch.int32).long()
    value, order = torch.sort(logits, dim=1, descending=True, stable=True)
    greedy = temperature <= 0
    t = torch.where(greedy, 1.0, temperature)[:, None]
    e = ((value - value[:, :1]) / t).exp()
    rank = torch.arange(e.shape[1], device="cuda")[None]
    within = rank < torch.where(greedy, 1, torch.where(top_k > 0, top_k, e.shape[1]))[:, None]
    mass = (e * within).cumsum(1)
    enough = (mass - e < top_p[:, None] * mass[:, -1:]) | (top_p >= 1)[:, None] | (rank == 0)
    keep = within & enough & (e >= min_p[:, None])
    weight = torch.zeros_like(e).scatter_(1, order, e * keep)
    running = weight.cumsum(1)
    token = (running > u[:, None] * running[:, -1:]).to(torch.uint8).argmax(1)
    chance = weight.gather(1, token[:, None])[:, 0] / running[:, -1]
    return {"token": token.to(torch.int32), "probability": chance.float()}


# ---- what a pass cannot do without ----

def work(case):
    if case["op"] == "sample":
        return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 7), "flops": 0.0}
    cached, added = _lengths(case)
    if case["op"] == "plan":
        page = case["page"]
        tokens = sum(max(a, 0) for a in added)
        moved = sum(_pages(c, page) if a < 0 else _pages(c + a, page) - _pages(c, page) for c, a in zip(cached, added))
        return {"bytes": 4.0 * (4 * len(cached) + 2 * moved + 2 * tokens), "flops": 0.0}
    tokens, heads = sum(added), case["heads"]
    pairs = sum(a * c + a * (a + 1) / 2 for c, a in zip(cached, added))
    rows = 2.0 * tokens * heads * (WIDTH + RANK)
    return {"bytes": 2.0 * WIDTH * (sum(cached) + tokens) + rows, "flops": 2.0 * pairs * heads * (WIDTH + RANK)}


# ---- the same in 64 bits, from the definitions ----

def _exact_plan(case, p):
    page, pages = case["page"], p["pages"]
    cached, added, table, ring = (p[k].tolist() for k in ("cached", "added", "table", "ring"))
    head, free = p["queue"].tolist()
    give = head + free
    lengths, starts, positions, slots, taken, released = [], [0], [], [], 0, 0
    for r, (c, a) in enumerate(zip(cached, added)):
        lengths.append(0 if a < 0 else c + a)
        starts.append(starts[-1] + max(a, 0))
        if a < 0:
            for k in range(_pages(c, page)):
                ring[give % pages] = table[r][k]
                give, released = give + 1, released + 1
        for position in range(c, c + max(a, 0)):
            if position % page == 0:
                table[r][position // page] = ring[(head + taken) % pages]
                taken += 1
            positions.append(position)
            slots.append(table[r][position // page] * page + position % page)
    pad = p["tokens"] - len(slots)
    return {"lengths": lengths, "starts": starts, "positions": positions + [0] * pad, "slots": slots + [-1] * pad,
            "queue": [(head + taken) % pages, free - taken + released], "info": [0, starts[-1], taken, released],
            "table": table, "ring": ring}


def _exact_attention(case, p):
    y = torch.empty((p["tokens"], case["heads"], RANK), dtype=torch.float64, device="cuda")
    starts, lengths = p["starts"].tolist(), p["lengths"].tolist()
    for r, n in enumerate(lengths):
        begin, end = starts[r], starts[r + 1]
        rows = p["pool"][p["table"][r, :_pages(n, case["page"])].long()].reshape(-1, WIDTH)[:n].double()
        after = torch.arange(n, device="cuda")[None] > torch.arange(n - (end - begin), n, device="cuda")[:, None]
        for h in range(case["heads"]):
            scores = (p["q"][begin:end, h].double() @ rows.T) * SCALE
            y[begin:end, h] = torch.softmax(scores.masked_fill(after, -math.inf), dim=-1) @ rows[:, :RANK]
    return {"y": y}


def _exact_sample(p):
    tokens, chances = [], []
    params, u = p["params"].cpu(), p["u"].double().tolist()
    for row, (logits, setting) in enumerate(zip(p["logits"], params)):
        temperature, top_p, min_p = (float(setting[k]) for k in (0, 2, 3))
        top_k = int(setting[1:2].view(torch.int32))
        x = logits.double().cpu()
        if temperature <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            chances.append(1.0)
            continue
        order = torch.from_numpy(np.argsort(-x.numpy(), kind="stable"))  # equal logits by index
        e = torch.exp((x[order] - x.max()) / temperature)
        keep = min(top_k, e.numel()) if top_k > 0 else e.numel()
        if top_p < 1:
            before = torch.cumsum(e[:keep], 0) - e[:keep]
            keep = max(1, min(keep, int((before < top_p * e[:keep].sum()).sum())))
        keep = max(1, min(keep, int((e >= min_p).sum())))
        kept, at = torch.sort(order[:keep])
        running = torch.cumsum(e[at], 0)
        k = min(int((running <= u[row] * running[-1]).sum()), keep - 1)
        tokens.append(int(kept[k]))
        chances.append(float(e[at[k]] / running[-1]))
    return {"token": torch.tensor(tokens), "probability": torch.tensor(chances, dtype=torch.float64)}


def exact(case, seed):
    p = _inputs(case, seed)
    if case["op"] == "plan":
        return {k: torch.tensor(v, dtype=torch.int32) for k, v in _exact_plan(case, p).items()}
    return _exact_attention(case, p) if case["op"] == "attention" else _exact_sample(p)
