"""What is timed of decoding with weights in 4 bits: bringing a bf16 matrix into that form, reading it back, products of
a few rows with it, and the log probabilities of the logits that such a model answers with.

A group of 32, 64 or 128 consecutive weights w of a row is held as e2m1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign) of
w / s and one bf16 scale s, the nearest to max |w| / 6 and at least 2^-126. Codes lie in tiles of 16 rows and 128 columns,
[rows / 16][cols / 128][4 q][16 rows][4 s][4 b] bytes, byte b holding columns 32 s + 8 q + 2 b (low nibble) and the next;
scales [rows / 16][cols / 128][16 rows][128 / group]. Rows and columns past the matrix are held as weights of 0.

Ops:
  store     a bf16 matrix into 4 bits, and what they stand for back as bf16
  read      a matrix in 4 bits as bf16
  product   y = x w^T of a few rows x: bf16 or f32 out, or silu(gate) up of a packed [gate; up] matrix
  logprobs  per row of logits: log probabilities of given tokens, entropy, and the top alternatives

Where own is true, run's calls are on the framework's own stream and wait for nothing: prepare's work is done when it returns,
and outputs are read after torch.cuda.synchronize() or gpu().sync().
"""
import math
import os
import sys

import torch

own = False

TILE, WIDE = 16, 128  # rows and columns of a tile of codes
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
NONE = -1  # the id (0xFFFFFFFF) of an alternative that is not there
CHUNK = 8192  # rows of a matrix that the plain forms take at a time


def listed():
    return [
        # An adapter's or a small model's odd matrix when it is loaded.
        {"name": "store_1000", "op": "store", "rows": 1000, "cols": 1096, "group": 32},
        # The largest projection of an 8B layer when a checkpoint is loaded.
        {"name": "store_gate_up", "op": "store", "rows": 24576, "cols": 4096, "group": 128},
        # A small layer's projection read back before a prompt's pass.
        {"name": "read_qkv", "op": "read", "rows": 4096, "cols": 1024, "group": 64},
        # A large layer's projection for a prompt's pass.
        {"name": "read_gate_up", "op": "read", "rows": 51200, "cols": 5120, "group": 32},
        # One token's projection in a small model: a launch's latency.
        {"name": "one_qkv", "op": "product", "n": 1, "rows": 4096, "cols": 1024, "group": 128, "out": "bf16"},
        # One token's gate and up projection in an 8B layer, the decode step's largest read.
        {"name": "one_gate_up", "op": "product", "n": 1, "rows": 24576, "cols": 4096, "group": 64, "out": "swiglu"},
        # One token's logits.
        {"name": "one_head", "op": "product", "n": 1, "rows": 151936, "cols": 4096, "group": 128, "out": "f32"},
        # A batch of conversations through a large layer's down projection.
        {"name": "batch_down", "op": "product", "n": 16, "rows": 5120, "cols": 25600, "group": 32, "out": "bf16"},
        # A short prompt, or drafted tokens of a batch, through a matrix of uneven size.
        {"name": "rows_61", "op": "product", "n": 61, "rows": 6150, "cols": 4104, "group": 32, "out": "f32"},
        # A chat's token with its 20 alternatives.
        {"name": "logprobs_one", "op": "logprobs", "rows": 1, "vocab": 151936, "stride": 151936, "type": "f32", "tokens": 1,
         "top": 20, "scale": 1.0},
        # Multiple choice: a batch's next-token logits in bf16, an odd vocabulary, masked entries, a temperature.
        {"name": "logprobs_choice", "op": "logprobs", "rows": 61, "vocab": 32001, "stride": 32001, "type": "bf16", "tokens": 4,
         "top": 5, "scale": 1.25},
        # Scoring a prompt: each position's next token.
        {"name": "logprobs_score", "op": "logprobs", "rows": 512, "vocab": 151936, "stride": 151936, "type": "f32", "tokens": 1,
         "top": 1, "scale": 1.0},
    ]


def log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "read", "product", "product", "product", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = log_uniform(rng, 100, 200000)
        return {"op": op, "rows": log_uniform(rng, 1, max(1, min(2048, 70000000 // vocab))), "vocab": vocab,
                "stride": vocab + rng.choice([0, 0, 3, 64]), "type": rng.choice(["f32", "bf16"]),
                "tokens": rng.choice([0, 1, 1, 2, 7]), "top": rng.choice([0, 1, 5, 20, 64]), "scale": rng.choice([1.0, 1.0, 0.5, 1.5])}
    # At most the work of the largest listed case of the op.
    n = log_uniform(rng, 1, 96) if op == "product" else 1
    most = {"store": 140000000, "read": 250000000, "product": min(600000000, 2000000000 // n)}[op]
    rows = log_uniform(rng, 1, 32768)
    case = {"op": op, "rows": rows, "cols": 8 * log_uniform(rng, 1, min(2048, most // (8 * rows))), "group": rng.choice([32, 64, 128])}
    if op == "product":
        case |= {"n": n, "out": rng.choice(["bf16", "f32", "swiglu"])}
        if case["out"] == "swiglu":
            case["rows"] = -(-rows // 32) * 32
    return case


# -- the form in 4 bits --

def up_to(n, m):
    return -(-n // m) * m


def quantise(w, group):
    """Codes (one to an element) and scales of rows of bf16 weights whose columns fill whole tiles."""
    x = w.float().unflatten(-1, (-1, group))
    top = x.abs().amax(-1)
    s = (top.double() / 6.0).float().bfloat16().float().clamp(min=2.0 ** -126)
    s = torch.where(top.isfinite(), s, math.nan)
    a, t = x.abs(), s[..., None]
    # 2 or 3 significant bits times a scale of 8, and a weight of 8: the comparisons are exact.
    code = (a > 0.25 * t).to(torch.uint8)
    for middle, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= middle * t) if up else (a > middle * t)
    code += 8 * ((x < 0) & (code > 0)).to(torch.uint8)
    return code.flatten(-2), s.bfloat16()


def pack(code, s):
    """Codes [rows][cols] and scales [rows][cols / group] of whole tiles as they lie."""
    c = code.view(-1, TILE, code.shape[1] // WIDE, 4, 4, 4, 2)  # [panel][row][tile][s][q][b][nibble]
    c = (c[..., 0] | c[..., 1] << 4).permute(0, 2, 4, 1, 3, 5)
    return c.reshape(-1), s.view(-1, TILE, c.shape[1], s.shape[1] // c.shape[1]).transpose(1, 2).reshape(-1)


def unpack(codes, scales, rows, cols, group):
    """What codes and scales of whole tiles stand for, [rows][cols] in 32 bits."""
    c = codes.view(rows // TILE, cols // WIDE, 4, TILE, 4, 4).permute(0, 3, 1, 4, 2, 5)
    c = torch.stack([c & 15, c >> 4], -1).reshape(rows, cols).to(torch.int32)
    values = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)[c]
    s = scales.view(rows // TILE, cols // WIDE, TILE, WIDE // group).transpose(1, 2).reshape(rows, cols // group)
    return (values.unflatten(-1, (-1, group)) * s.float()[..., None]).flatten(-2)


def chunks(case):
    """(first row, rows behind the last, their panels' share of codes and of scales) of the matrix, CHUNK rows at a time."""
    wide = up_to(case["cols"], WIDE)
    for first in range(0, case["rows"], CHUNK):
        last = min(first + CHUNK, up_to(case["rows"], TILE))
        yield (first, min(last, case["rows"]), slice(first * wide // 2, last * wide // 2),
               slice(first * (wide // case["group"]), last * (wide // case["group"])))


def padded(w):
    """Rows of weights with zeros up to whole tiles."""
    out = w.new_zeros((up_to(w.shape[0], TILE), up_to(w.shape[1], WIDE)))
    out[:w.shape[0], :w.shape[1]] = w
    return out


# -- inputs --

def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def weights(g, rows, cols):
    """bf16 weights as a trained matrix has them: normal, rows of uneven size, a few far values."""
    w = torch.randn((rows, cols), device="cuda", generator=g) * 0.02
    w *= 0.5 + torch.rand((rows, 1), device="cuda", generator=g)
    w *= torch.where(torch.rand((rows, cols), device="cuda", generator=g) < 0.001, 6.0, 1.0)
    return w.bfloat16()


def held(case, g):
    """A matrix in 4 bits."""
    whole = up_to(case["rows"], TILE) * up_to(case["cols"], WIDE)
    state = {"codes": torch.empty(whole // 2, dtype=torch.uint8, device="cuda"),
             "scales": torch.empty(whole // case["group"], dtype=torch.bfloat16, device="cuda")}
    for first, last, of_codes, of_scales in chunks(case):
        state["codes"][of_codes], state["scales"][of_scales] = pack(*quantise(padded(weights(g, last - first, case["cols"])),
                                                                              case["group"]))
    return state


def prepare(case, seed):
    g = generator(seed)
    state = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab, stride = case["rows"], case["vocab"], case["stride"]
        # Logits as a head gives them: most of a row far below a few; every eighth row with most tokens masked.
        x = torch.randn((rows, stride), device="cuda", generator=g) * 2.5
        x[torch.rand((rows, stride), device="cuda", generator=g) < 3.0 / vocab] += 12.0
        x[7::8].masked_fill_(torch.rand((rows, stride), device="cuda", generator=g)[7::8] < 0.9, -math.inf)
        x[:, 0] = x[:, 0].clamp(min=-20.0)
        state["logits"] = x.to(torch.bfloat16 if case["type"] == "bf16" else torch.float32)
        state["tokens"] = torch.randint(0, vocab, (rows, case["tokens"]), device="cuda", generator=g, dtype=torch.int32)
        state |= {"token_lp": torch.zeros((rows, case["tokens"]), device="cuda"), "entropy": torch.zeros(rows, device="cuda"),
                  "top_ids": torch.zeros((rows, case["top"]), dtype=torch.int32, device="cuda"),
                  "top_lp": torch.zeros((rows, case["top"]), device="cuda")}
    else:
        state |= held(case, g)
        rows, cols = case["rows"], case["cols"]
        if case["op"] == "product":
            x = torch.randn((case["n"], cols), device="cuda", generator=g)
            x *= torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 20.0, 1.0)
            state["x"] = x.bfloat16()
            state["y"] = torch.zeros((case["n"], rows // 2 if case["out"] == "swiglu" else rows), device="cuda",
                                     dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)
        else:
            state["w"] = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
            if case["op"] == "store":
                state["from"] = weights(g, rows, cols)
    if own:
        state["call"] = call_of(state)
    return state


# -- the framework's calls --

_kept = {}


def gpu():
    """The program's one device handle."""
    if "gpu" not in _kept:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x0ne-engine_amd"))
        from x0ne_core import Gpu
        _kept["gpu"] = Gpu()
    return _kept["gpu"]


def call_of(state):
    """What the program keeps of a matrix in 4 bits, or of a sampler's buffers: their descriptor and workspace. torch's own work
    on the inputs is done behind it, as the calls are on another stream."""
    case, g = state["case"], gpu()
    from x0ne_core import LogProbs, W4
    at = {k: v.data_ptr() if v.numel() else 0 for k, v in state.items() if isinstance(v, torch.Tensor)}
    if case["op"] != "logprobs":
        torch.cuda.synchronize()
        return W4(codes=at["codes"], scales=at["scales"], rows=case["rows"], cols=case["cols"], group=case["group"])
    d = LogProbs(logits=at["logits"], stride=case["stride"], tokens=at["tokens"], token_lp=at["token_lp"], entropy=at["entropy"],
                 top_ids=at["top_ids"], top_lp=at["top_lp"], rows=case["rows"], vocab=case["vocab"], per_row=case["tokens"],
                 top=case["top"], bf16=case["type"] == "bf16", scale=case["scale"])
    size = g.logprobs_work_bytes(d)
    state["work"] = torch.zeros(max(size, 1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    d.work, d.work_bytes = state["work"].data_ptr(), size
    return d


def run_own(state):
    g, case = gpu(), state["case"]
    if "call" not in state:
        state["call"] = call_of(state)
    call = state["call"]
    if case["op"] == "store":
        g.w4_quantise(call, state["from"].data_ptr())
        g.w4_read(call, state["w"].data_ptr())
    elif case["op"] == "read":
        g.w4_read(call, state["w"].data_ptr())
    elif case["op"] == "product":
        g.w4_gemv(call, state["x"].data_ptr(), case["n"], state["y"].data_ptr(), case["out"])
    else:
        g.logprobs(call)


# -- the plain form --

def plain_store(state):
    case = state["case"]
    for first, last, of_codes, of_scales in chunks(case):
        state["codes"][of_codes], state["scales"][of_scales] = pack(*quantise(padded(state["from"][first:last]), case["group"]))


def values(state):
    """Rows of the matrix in 32 bits, CHUNK at a time."""
    case = state["case"]
    for first, last, of_codes, of_scales in chunks(case):
        w = unpack(state["codes"][of_codes], state["scales"][of_scales], up_to(last - first, TILE), up_to(case["cols"], WIDE),
                   case["group"])
        yield first, last, w[:last - first, :case["cols"]]


def plain_read(state):
    for first, last, w in values(state):
        state["w"][first:last] = w.bfloat16()


def plain_product(state):
    case, x = state["case"], state["x"].float()
    y = torch.empty((case["n"], case["rows"]), device="cuda")
    for first, last, w in values(state):
        y[:, first:last] = x @ w.t()
    if case["out"] == "swiglu":
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    state["y"].copy_(y)


def plain_logprobs(state):
    case = state["case"]
    raw = state["logits"][:, :case["vocab"]].float()
    x = raw * case["scale"]
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    # A row with NaN, infinity or nothing but -infinity has no distribution: NaN throughout.
    state["entropy"].copy_(torch.log(total[:, 0]) - torch.where(p > 0, p * (x - top), p).sum(-1) / total[:, 0])
    lse = top + torch.log(total)
    state["token_lp"].copy_(torch.gather(x, 1, state["tokens"].long()) - lse)
    if case["top"] == 0:
        return
    best, ids = torch.sort(raw, dim=-1, descending=True, stable=True)
    best, ids = best[:, :case["top"]], ids[:, :case["top"]]
    there = (best > -math.inf) & total.isfinite()
    state["top_ids"].fill_(NONE)
    state["top_lp"].fill_(-math.inf)
    state["top_ids"][:, :ids.shape[1]] = torch.where(there, ids, NONE).int()
    state["top_lp"][:, :ids.shape[1]] = best * case["scale"] - lse
    state["top_lp"] += total - total


def run(state):
    op = state["case"]["op"]
    if own:
        run_own(state)
    elif op == "store":
        plain_store(state)
        plain_read(state)
    else:
        {"read": plain_read, "product": plain_product, "logprobs": plain_logprobs}[op](state)
    if op == "store":
        return {"w": state["w"], "scales": state["scales"]}
    if op == "read":
        return {"w": state["w"]}
    if op == "product":
        return {"y": state["y"]}
    out = {"entropy": state["entropy"]}
    if state["case"]["tokens"]:
        out["token_lp"] = state["token_lp"]
    if state["case"]["top"]:
        out |= {"top_ids": state["top_ids"], "top_lp": state["top_lp"]}
    return out


# -- what a pass cannot do without --

def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        each = 4 + 8 * case["tokens"] + 8 * case["top"]
        return {"bytes": n * (2 if case["type"] == "bf16" else 4) + case["rows"] * each, "flops": 6 * n}
    n = case["rows"] * case["cols"]
    codes = n // 2 + 2 * case["rows"] * -(-case["cols"] // case["group"])
    if case["op"] == "store":
        return {"bytes": 4 * n + codes, "flops": 4 * n}
    if case["op"] == "read":
        return {"bytes": 2 * n + codes, "flops": n}
    out = {"bf16": 2, "f32": 4, "swiglu": 1}[case["out"]]
    return {"bytes": codes + case["n"] * (2 * case["cols"] + out * case["rows"]), "flops": 2 * n * case["n"]}


# -- the same in 64 bits, from the definition --

def power(e):
    """2^e of whole numbers, from the bits."""
    return (e.long() + 1023 << 52).view(torch.float64)


def exact_scales(w, group):
    """The bf16 nearest to max |w| / 6 of each group, in 64 bits: 8 bits of the value, the even ones where two are as near."""
    top = w.abs().unflatten(-1, (-1, group)).amax(-1) / 6.0
    _, e = torch.frexp(top)
    unit = power(e - 8)
    return torch.clamp(torch.where(top > 0, torch.round(top / unit) * unit, 0.0), min=2.0 ** -126)


def exact_store(s, case):
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    values, scales = [], []
    for first, last, _, _ in chunks(case):
        w = padded(s["from"][first:last]).double()
        sc = exact_scales(w, case["group"])
        each = sc.repeat_interleave(case["group"], -1)
        q = w.abs() / each
        hi = torch.searchsorted(grid, q.contiguous()).clamp(1, 7)
        below, above = q - grid[hi - 1], grid[hi] - q
        code = torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)
        values.append((torch.sign(w) * grid[code] * each)[:last - first, :case["cols"]])
        per = WIDE // case["group"]
        scales.append(sc.reshape(-1, TILE, w.shape[1] // WIDE, per).permute(0, 2, 1, 3).reshape(-1))
    return {"w": torch.cat(values), "scales": torch.cat(scales)}


def exact_rows(s, case, first, last):
    """Rows of a matrix in 4 bits, element by element from the definition of where it lies."""
    cols, wide = case["cols"], up_to(case["cols"], WIDE)
    r = torch.arange(first, last, device="cuda")[:, None]
    c = torch.arange(cols, device="cuda")[None]
    tile, k = (r // TILE) * (wide // WIDE) + c // WIDE, c % WIDE
    byte = s["codes"][tile * 1024 + (k // 8 % 4) * 256 + (r % TILE) * 16 + (k // 32) * 4 + k % 8 // 2].int()
    code = torch.where(k % 2 == 1, byte // 16, byte % 16)
    m = code % 8
    value = torch.where(m < 2, m / 2.0, (1.0 + m % 2 / 2.0) * power(m // 2 - 1))
    per = WIDE // case["group"]
    scale = s["scales"][(tile * TILE + r % TILE) * per + k // case["group"]].double()
    return torch.where(code > 7, -value, value) * scale


def exact_product(s, case):
    x = s["x"].double()
    y = torch.cat([x @ exact_rows(s, case, i, min(i + CHUNK, case["rows"])).t().contiguous()
                   for i in range(0, case["rows"], CHUNK)], -1)
    if case["out"] == "swiglu":
        half = case["rows"] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return {"y": y}


def exact_logprobs(s, case):
    x = s["logits"][:, :case["vocab"]].double()
    lp = torch.log_softmax(x * case["scale"], -1)
    out = {"entropy": -torch.where(lp > -math.inf, lp * torch.exp(lp), 0.0).sum(-1)}
    if case["tokens"]:
        out["token_lp"] = torch.stack([lp[torch.arange(case["rows"], device="cuda"), s["tokens"][:, j].long()]
                                       for j in range(case["tokens"])], 1)
    if case["top"]:
        ids = torch.full((case["rows"], case["top"]), NONE, dtype=torch.int64, device="cuda")
        best = torch.full((case["rows"], case["top"]), -math.inf, dtype=torch.float64, device="cuda")
        left, at = x.clone(), torch.arange(case["rows"], device="cuda")
        for j in range(min(case["top"], case["vocab"])):
            most = left.amax(-1)
            first = (left == most[:, None]).int().argmax(-1)
            ids[:, j] = torch.where(most > -math.inf, first, NONE)
            best[:, j] = torch.where(most > -math.inf, lp[at, first], -math.inf)
            left[at, first] = -math.inf
        out |= {"top_ids": ids, "top_lp": best}
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read":
        return {"w": torch.cat([exact_rows(s, case, i, min(i + CHUNK, case["rows"])) for i in range(0, case["rows"], CHUNK)])}
    return {"store": exact_store, "product": exact_product, "logprobs": exact_logprobs}[case["op"]](s, case)
