"""The products of 8-bit floating point that the FFN's experts take, as measurable cases.

Kinds:
  quantize   rows, or a matrix of weights, in e4m3 with one scale to a block of 1 x 128 or 128 x 128
             (lm_fp8_quantize)
  gemm       the product of such rows with such a matrix (lm_fp8_gemm)
  grouped    the same with a matrix for each expert and ragged groups of rows (lm_fp8_grouped_gemm)
  swiglu     the experts' gate and up products, their SwiGLU, and its rows in e4m3 blocks again
             (lm_fp8_grouped_swiglu)

Sizes are DeepSeek-V2's and V2-Lite's: hidden 2048 and 5120, experts of 1408 and 1536 channels, 64 and 160 of them of
which a token takes 6, a dense FFN of 10944, an output projection of 16384 channels (and other ones).
"""
import math
import random

import torch

own = False  # False: elementary torch operations; True: litemind_amd's operators

BLOCK = 128
LARGEST = 448.0        # of e4m3
LEAST = 2.0 ** -126    # the least scale
E4M3 = torch.float8_e4m3fn
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---- cases ----

def _quantize(rows, width, dtype, block_rows=1, pad=0):
    return {"op": "quantize", "rows": rows, "width": width, "dtype": dtype, "block_rows": block_rows, "pad": pad}


def _gemm(rows, out, inner, dtype):
    return {"op": "gemm", "rows": rows, "out": out, "inner": inner, "dtype": dtype}


def _experts(op, tokens, experts, out, inner, dtype="fp32", skewed=False, mix=1):
    return {"op": op, "tokens": tokens, "experts": experts, "top_k": min(6, experts), "out": out, "inner": inner,
            "dtype": dtype, "skewed": skewed, "mix": mix}


def listed():
    def named(name, case):
        return {"name": name, **case}

    return [
        # one token's hidden state, before its products: the smallest call, latency counts
        named("quantize_token", _quantize(1, 2048, "fp32")),
        # the hidden states of a long prompt
        named("quantize_prompt", _quantize(2047, 5120, "fp32")),
        # the dense layer's down projection when it is loaded: an odd last block
        named("quantize_weights", _quantize(2048, 10944, "bf16", block_rows=128)),
        # one token through the dense layer's down projection: the reduced axis is long, its last block is half full
        named("gemm_token", _gemm(1, 2048, 10944, "fp32")),
        # a decode step of 48 conversations through the dense layer's up projection
        named("gemm_batch", _gemm(48, 10944, 2048, "bf16")),
        # a prompt through the larger model's output projection: the most products
        named("gemm_prompt", _gemm(2048, 5120, 16384, "bf16")),
        # one token's six experts, down projection
        named("grouped_token", _experts("grouped", 1, 64, 2048, 1408)),
        # a decode step of 61 conversations: a few rows to an expert, nearly all experts
        named("grouped_batch", _experts("grouped", 61, 64, 2048, 1408, "fp16", mix=2)),
        # a prompt whose tokens prefer a few experts
        named("grouped_prompt", _experts("grouped", 2048, 64, 2048, 1408, skewed=True, mix=3)),
        # one token's six experts, gate and up
        named("swiglu_token", _experts("swiglu", 1, 64, 1408, 2048, mix=4)),
        # a decode step of 32 conversations over the larger model's 160 experts: the most weights
        named("swiglu_wide_batch", _experts("swiglu", 32, 160, 1536, 5120, mix=5)),
        # a prompt whose tokens prefer a few experts, gate and up
        named("swiglu_prompt", _experts("swiglu", 2048, 64, 1408, 2048, skewed=True, mix=6)),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "grouped", "grouped", "grouped", "swiglu", "swiglu", "swiglu"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "quantize":
        width = rng.choice([1408, 1536, 2048, 2816, 5120, 10944, _log_uniform(rng, 1, 16384)])
        if rng.random() < 0.3:
            return _quantize(_log_uniform(rng, 100, 12288), width, "bf16", block_rows=BLOCK)
        return _quantize(_log_uniform(rng, 1, 4096), width, dtype, pad=rng.choice([0, 0, 8, 33]))
    if op == "gemm":
        inner = rng.choice([1408, 1536, 2048, 5120, 10944, 16384, 16 * _log_uniform(rng, 1, 1024)])
        out = rng.choice([2048, 2816, 5120, 10944, _log_uniform(rng, 1, 24576)])
        return _gemm(_log_uniform(rng, 1, max(1, min(4096, (1 << 37) // (out * inner)))), out, inner, dtype)
    experts = rng.choice([64, 64, 160, rng.choice([2, 5, 8, 16, 32])])
    hidden, inter = (5120, 1536) if experts == 160 else rng.choice([(2048, 1408), (2048, 1408), (1024, 16 * _log_uniform(rng, 4, 128))])
    out, inner = (hidden, inter) if op == "grouped" else (inter, hidden)
    tokens = _log_uniform(rng, 1, 512 if experts == 160 else 2048)
    return _experts(op, tokens, experts, out, inner, dtype if op == "grouped" else "fp32", rng.random() < 0.5,
                    rng.randrange(1, 1 << 30))


# ---- inputs, from the seed alone (which experts a token takes: from the case alone) ----

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 41)
    return g


def _blocks(n):
    return -(-n // BLOCK)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _to_blocks(x, block_rows):
    """e4m3 codes and scales of x [..., rows, width], as a model's weights and rows come."""
    rows, width = x.shape[-2:]
    tall, wide = -(-rows // block_rows), _blocks(width)
    x = torch.nn.functional.pad(x.float(), (0, wide * BLOCK - width, 0, tall * block_rows - rows))
    x = x.view(*x.shape[:-2], tall, block_rows, wide, BLOCK)
    scale = (x.abs().amax((-3, -1)) / LARGEST).clamp(min=LEAST)
    q = (x * (1.0 / scale)[..., :, None, :, None]).to(E4M3)
    q = q.reshape(*q.shape[:-4], tall * block_rows, wide * BLOCK).view(torch.uint8)[..., :rows, :width]
    return q.contiguous(), scale.contiguous()


def _route(case):
    """First row of each expert's group, and the assignment token * top_k + rank of each row, expert by expert."""
    g = torch.Generator()
    g.manual_seed(case["mix"])
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    score = torch.rand((T, E), generator=g).log().neg().log().neg()
    if case["skewed"]:
        liked = torch.randperm(E, generator=g)[:max(1, E // 8)]
        score[:, liked] += 3.0
    expert = score.topk(k, dim=1).indices.reshape(-1)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(expert, minlength=E).cumsum(0)
    return offsets, torch.argsort(expert, stable=True).to(torch.int32)


def _inputs(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "quantize":
        rows, width = case["rows"], case["width"]
        x = _randn(g, rows, width + case["pad"]) * (0.02 if case["block_rows"] > 1 else 1.0)
        if case["block_rows"] == 1:  # a few channels are far larger than the others
            x[:, torch.randint(0, width, (1 + width // 300,), generator=g, device="cuda")] *= 20.0
        return {"x": x.to(DTYPES[case["dtype"]])}
    out, inner = case["out"], case["inner"]
    if op == "gemm":
        a, a_scale = _to_blocks(_randn(g, case["rows"], inner), 1)
        w, w_scale = _to_blocks(_randn(g, out, inner) * 0.02, BLOCK)
        return {"a": a, "a_scale": a_scale, "w": w, "w_scale": w_scale}
    E, rows = case["experts"], case["tokens"] * case["top_k"]
    parts = 2 if op == "swiglu" else 1
    # the gate and up products read the tokens, the down product a row of each assignment
    a, a_scale = _to_blocks(_randn(g, case["tokens"] if op == "swiglu" else rows, inner), 1)
    w = torch.empty((E, parts, out, inner), dtype=torch.uint8, device="cuda")
    w_scale = torch.empty((E, parts, _blocks(out), _blocks(inner)), device="cuda")
    for e in range(E):
        w[e], w_scale[e] = _to_blocks(_randn(g, parts, out, inner) * 0.03, BLOCK)
    offsets, perm = _route(case)
    return {"a": a, "a_scale": a_scale, "w": w, "w_scale": w_scale, "offsets": offsets.cuda(), "perm": perm.cuda(),
            "most": int((offsets[1:] - offsets[:-1]).max()), "active": torch.nonzero(offsets[1:] > offsets[:-1])[:, 0].cuda()}


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
        self.dtype = {"fp32": lm.DT_F32, "fp16": lm.DT_F16, "bf16": lm.DT_BF16}[case["dtype"]]
        if op == "quantize":
            rows, width, tall = case["rows"], case["width"], -(-case["rows"] // case["block_rows"])
            self.q = torch.zeros((rows, width), dtype=torch.uint8, device="cuda")
            self.scale = torch.zeros((tall, _blocks(width)), device="cuda")
        else:
            rows = case["rows"] if op == "gemm" else case["tokens"] * case["top_k"]
            if op == "swiglu":
                self.q = torch.zeros((rows, case["out"]), dtype=torch.uint8, device="cuda")
                self.scale = torch.zeros((rows, _blocks(case["out"])), device="cuda")
            else:
                self.y = torch.zeros((rows, case["out"]), dtype=DTYPES[case["dtype"]], device="cuda")
            if op != "gemm":
                self.groups = lm.Fp8Groups(groups=case["experts"], rows=rows, offsets=p["offsets"].data_ptr())
                if op == "swiglu":  # row i reads the token of its assignment
                    self.groups.source, self.groups.divisor = p["perm"].data_ptr(), case["top_k"]
                else:  # row i is written to its assignment's place
                    self.groups.target = p["perm"].data_ptr()
        torch.cuda.synchronize()

    def __del__(self):
        if getattr(self, "ctx", None) is not None and self.ctx.handle:
            self.ctx.synchronize()
            self.ctx.close()


def prepare(case, seed):
    return State(case, seed)


# ---- one pass ----

def run(s):
    c, p, op = s.case, s.p, s.case["op"]
    if not own:
        return {"quantize": _plain_quantize, "gemm": _plain_gemm, "grouped": _plain_grouped, "swiglu": _plain_swiglu}[op](c, p)
    if op == "quantize":
        s.ctx.fp8_quantize(p["x"].data_ptr(), c["rows"], c["width"], s.q.data_ptr(), s.scale.data_ptr(), dtype=s.dtype,
                           row_stride=c["width"] + c["pad"], block_rows=c["block_rows"])
        return {"q": s.q.view(E4M3), "scale": s.scale}
    if op == "gemm":
        s.ctx.fp8_gemm(p["a"].data_ptr(), p["a_scale"].data_ptr(), c["rows"], p["w"].data_ptr(), p["w_scale"].data_ptr(),
                       c["out"], c["inner"], s.y.data_ptr(), dtype=s.dtype)
        return {"y": s.y}
    if op == "grouped":
        s.ctx.fp8_grouped_gemm(s.groups, p["a"].data_ptr(), p["a_scale"].data_ptr(), p["a"].shape[0], p["w"].data_ptr(),
                               p["w_scale"].data_ptr(), c["out"], c["inner"], s.y.data_ptr(), s.y.shape[0], dtype=s.dtype)
        return {"y": s.y}
    s.ctx.fp8_grouped_swiglu(s.groups, p["a"].data_ptr(), p["a_scale"].data_ptr(), p["a"].shape[0], p["w"].data_ptr(),
                             p["w_scale"].data_ptr(), c["out"], c["inner"], s.q.data_ptr(), s.scale.data_ptr())
    return {"q": s.q.view(E4M3), "scale": s.scale}


def _plain_blocks(x, block_rows):
    """x [rows, width] fp32 in e4m3 blocks."""
    rows, width = x.shape
    tall, wide = -(-rows // block_rows), _blocks(width)
    padded = torch.zeros((tall * block_rows, wide * BLOCK), device=x.device)
    padded[:rows, :width] = x
    padded = padded.view(tall, block_rows, wide, BLOCK)
    scale = (padded.abs().amax((1, 3)) / LARGEST).clamp(min=LEAST)
    q = (padded * (1.0 / scale)[:, None, :, None]).to(E4M3).view(torch.uint8)
    return {"q": q.reshape(tall * block_rows, wide * BLOCK)[:rows, :width].contiguous().view(E4M3), "scale": scale}


def _plain_quantize(case, p):
    return _plain_blocks(p["x"][:, :case["width"]].float(), case["block_rows"])


def _wide(q, scale, block_rows):
    """The fp32 values of e4m3 blocks [..., rows, width]."""
    rows, width = q.shape[-2:]
    each = scale.repeat_interleave(block_rows, -2)[..., :rows, :] if block_rows > 1 else scale
    return q.view(E4M3).float().mul_(each.repeat_interleave(BLOCK, -1)[..., :width])


def _plain_gemm(case, p):
    y = _wide(p["a"], p["a_scale"], 1) @ _wide(p["w"], p["w_scale"], BLOCK).t()
    return {"y": y.to(DTYPES[case["dtype"]])}


def _by_expert(case, p, x, w):
    """Rows x [rows, inner] in expert order, times w [active experts, out, inner]: every group padded to the longest."""
    offsets = p["offsets"].long()
    first, count = offsets[p["active"]], (offsets[1:] - offsets[:-1])[p["active"]]
    i = torch.arange(p["most"], device="cuda")
    at = (first[:, None] + i[None]).clamp(max=x.shape[0] - 1)
    y = torch.bmm(x[at], w.transpose(1, 2).contiguous())
    return y[i[None] < count[:, None]]


def _plain_grouped(case, p):
    perm = p["perm"].long()
    w = _wide(p["w"][p["active"], 0], p["w_scale"][p["active"], 0], BLOCK)
    rows = _by_expert(case, p, _wide(p["a"], p["a_scale"], 1), w)
    return {"y": torch.empty_like(rows).index_copy_(0, perm, rows).to(DTYPES[case["dtype"]])}


def _plain_swiglu(case, p):
    x = _wide(p["a"], p["a_scale"], 1)[p["perm"].long() // case["top_k"]]
    gate, up = (_by_expert(case, p, x, _wide(p["w"][p["active"], part], p["w_scale"][p["active"], part], BLOCK))
                for part in (0, 1))
    return _plain_blocks(gate / (1.0 + (-gate).exp()) * up, 1)


# ---- what a pass cannot do without ----

def work(case):
    op = case["op"]
    if op == "quantize":
        rows, width = case["rows"], case["width"]
        return {"bytes": rows * width * (BYTES[case["dtype"]] + 1.0) + 4.0 * -(-rows // case["block_rows"]) * _blocks(width),
                "flops": 0.0}
    out, inner = case["out"], case["inner"]
    row, matrix = inner + 4.0 * _blocks(inner), float(out * inner) + 4.0 * _blocks(out) * _blocks(inner)
    if op == "gemm":
        rows = case["rows"]
        return {"bytes": rows * row + matrix + rows * out * BYTES[case["dtype"]], "flops": 2.0 * rows * out * inner}
    offsets, _ = _route(case)
    active, rows = int((offsets[1:] > offsets[:-1]).sum()), case["tokens"] * case["top_k"]
    if op == "grouped":
        return {"bytes": rows * (row + 4.0 + out * BYTES[case["dtype"]]) + active * matrix, "flops": 2.0 * rows * out * inner}
    return {"bytes": case["tokens"] * row + rows * (4.0 + out + 4.0 * _blocks(out)) + 2.0 * active * matrix,
            "flops": 4.0 * rows * out * inner}


# ---- the same in 64 bits, from the definitions ----

def _exact_blocks(x, block_rows):
    rows, width = x.shape
    q = torch.empty_like(x)
    scales = []
    for b in range(_blocks(width)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        most = part.abs().amax(1)
        if block_rows > 1:
            most = torch.stack([m.max() for m in most.split(block_rows)])
        s = torch.clamp(most / LARGEST, min=LEAST)
        scales.append(s)
        v = part / s.repeat_interleave(block_rows)[:rows, None]
        step = torch.exp2(torch.clamp(torch.frexp(v).exponent.double() - 1, min=-6) - 3)  # four bits, least 2^-9
        q[:, b * BLOCK:(b + 1) * BLOCK] = torch.clamp(torch.round(v / step) * step, -LARGEST, LARGEST)
    return {"q": q, "scale": torch.stack(scales, 1)}


def _exact_values(q, scale, block_rows):
    value = q.view(E4M3).double()
    rows = torch.arange(q.shape[-2], device="cuda") // block_rows
    return value * scale.double()[rows][:, torch.arange(q.shape[-1], device="cuda") // BLOCK]


def exact(case, seed):
    p, op = _inputs(case, seed), case["op"]
    if op == "quantize":
        return _exact_blocks(p["x"][:, :case["width"]].double(), case["block_rows"])
    a = _exact_values(p["a"], p["a_scale"], 1)
    if op == "gemm":
        return {"y": a @ _exact_values(p["w"], p["w_scale"], BLOCK).T}
    offsets, perm = p["offsets"].tolist(), p["perm"].long()
    y = torch.empty((perm.numel(), case["out"]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        group = slice(offsets[e], offsets[e + 1])
        rows = perm[group]
        if rows.numel() == 0:
            continue
        w = [_exact_values(q, s, BLOCK).T for q, s in zip(p["w"][e], p["w_scale"][e])]
        if op == "grouped":
            y[rows] = a[group] @ w[0]
        else:
            x = a[rows // case["top_k"]]
            gate = x @ w[0]
            y[group] = gate * torch.sigmoid(gate) * (x @ w[1])
    return {"y": y} if op == "grouped" else _exact_blocks(y, 1)
