"""What is timed of the 8-bit paged K/V cache: writing it, reading it back, decode attention over it, and decode
attention over the pages that a cheap score selects.

A cache row of 128 values x is held as e4m3 codes of x / 2^e and one byte e + 127, e the smallest exponent
(from -117 on) with 448 * 2^e >= max |x|. Codes are paged [pool][kv_heads][2][2048] (16 keys' rows, then the
values of 16 positions dim-major), scale bytes [pool][kv_heads][2][16]; page_table [seqs][seq_pages] names the
physical page of 16 positions. Bounds [pool][kv_heads][2][128] hold the smallest and the largest key value of each
dim of a complete page.

Ops:
  write   RMSNorm of each head of q and k, rotation by position, k and v quantised into their pages; the bounds of
          the pages that this completes
  read    positions below a sequence's length back as bf16 pages
  attend  one query token per sequence over its keys, sequences of different lengths
  sparse  pages chosen for each query and kv head by their bounds, then attention over those
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HEAD, HALF, PAGE = 128, 64, 16
EPS, THETA, SCALE = 1e-6, 1e6, float(np.float32(1.0 / math.sqrt(128.0)))
LOWEST = -117  # the smallest scale exponent: 2^-117 times e4m3's smallest step is bf16's smallest normal value


def listed():
    return [
        # A chat's decode step at the smallest model: one row, where a launch's latency is all.
        {"name": "write_one_row", "op": "write", "q_heads": 16, "kv_heads": 8, "seqs": 1, "rows": 1, "longest": 777},
        # A batched decode step: one row for each of 64 conversations, some of which complete a page.
        {"name": "write_batch_64", "op": "write", "q_heads": 32, "kv_heads": 8, "seqs": 64, "rows": 64, "longest": 2048},
        # Prompts of uneven lengths side by side, none starting at a page's start, the last rows padding.
        {"name": "write_prompts_777", "op": "write", "q_heads": 64, "kv_heads": 8, "seqs": 5, "rows": 777, "longest": 1500},
        # A prefill pass of a long document.
        {"name": "write_prompt_2048", "op": "write", "q_heads": 32, "kv_heads": 8, "seqs": 1, "rows": 2048, "longest": 8192},
        # A short conversation read back before its next prompt.
        {"name": "read_333", "op": "read", "kv_heads": 8, "seqs": 1, "longest": 333},
        # The prefixes of a batch of long conversations.
        {"name": "read_batch_8k", "op": "read", "kv_heads": 8, "seqs": 16, "longest": 8192},
        # A chat's decode step early on: latency.
        {"name": "attend_164", "op": "attend", "q_heads": 16, "kv_heads": 8, "seqs": 1, "longest": 164},
        # One user with a long document in the cache.
        {"name": "attend_32k", "op": "attend", "q_heads": 32, "kv_heads": 8, "seqs": 1, "longest": 32768},
        # A batch of conversations of all lengths, an empty slot among them.
        {"name": "attend_batch_16", "op": "attend", "q_heads": 32, "kv_heads": 8, "seqs": 16, "longest": 8192},
        # A full batch at the largest model: the cache's bytes.
        {"name": "attend_batch_64", "op": "attend", "q_heads": 64, "kv_heads": 8, "seqs": 64, "longest": 6000},
        # The long document again, through 128 of its 2048 pages.
        {"name": "sparse_32k", "op": "sparse", "q_heads": 32, "kv_heads": 8, "seqs": 1, "longest": 32768, "budget": 128},
        # A batch of long conversations, each through at most 1024 of its positions.
        {"name": "sparse_batch_16", "op": "sparse", "q_heads": 32, "kv_heads": 8, "seqs": 16, "longest": 16000, "budget": 64},
    ]


def log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "sparse"])
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16] if kv_heads < 8 else [1, 2, 3, 4, 8])
    if op == "write":
        seqs = log_uniform(rng, 1, 64)
        return {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "seqs": seqs,
                "rows": log_uniform(rng, seqs, max(seqs, 2048)), "longest": log_uniform(rng, 2049, 4096)}
    longest = log_uniform(rng, 1 if op != "sparse" else 64, 32768)
    seqs = log_uniform(rng, 1, max(1, min(64, 131072 // longest)))
    case = {"op": op, "kv_heads": kv_heads, "seqs": seqs, "longest": longest}
    if op != "read":
        case["q_heads"] = q_heads
    if op == "sparse":
        case["budget"] = log_uniform(rng, 2, 256)
    return case


# -- inputs --

def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def host(seed):
    return np.random.default_rng(seed)


def normal(g, shape):
    return torch.randn(shape, device="cuda", generator=g)


def pages_of(case):
    """Entries of a sequence's page table: its longest length and one page more."""
    return -(-case["longest"] // PAGE) + 1


def lengths(case):
    """Lengths spread evenly up to the longest; from 8 sequences on one slot of the batch is empty."""
    n = case["seqs"]
    lens = np.maximum(case["longest"] * np.arange(n, 0, -1) // n, 1)
    if n >= 8:
        lens[-1] = 0
    return lens


def write_rows(case, seed):
    """(sequence, position) of each row: runs of consecutive positions at the ends of the sequences; in runs of
    several rows the last sequence's are padding."""
    r, n, rows = host(seed + 1), case["seqs"], case["rows"]
    cuts = np.sort(r.choice(np.arange(1, rows), n - 1, replace=False)) if n > 1 else np.array([], np.int64)
    counts = np.diff(np.concatenate([[0], cuts, [rows]])).astype(np.int64)
    seq = np.repeat(np.arange(n), counts)
    first = np.array([r.integers(0, case["longest"] - c + 1) for c in counts])
    if n == 1 and rows > 1:
        first[0] -= first[0] % PAGE
    pos = np.concatenate([f + np.arange(c) for f, c in zip(first, counts)])
    if rows > n > 1:
        seq[seq == n - 1] = -1
    return seq, pos


def power(e):
    """2^e of whole numbers, from the bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def quantise(x):
    """The codes and scale bytes of rows of 128 values."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, torch.where(m > 0.875, e - 8, e - 9), LOWEST).clamp(min=LOWEST)
    return (x * power(-e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def values(codes, scales):
    """What code bytes and their rows' scale bytes stand for."""
    return codes.view(torch.float8_e4m3fn).float() * power(scales.to(torch.int32) - 127)


def key_values(state, pages):
    """Keys of pages [...], [..., kv_heads, 16, 128]."""
    codes = state["codes"][:, :, 0][pages].unflatten(-1, (PAGE, HEAD))
    return values(codes, state["scales"][:, :, 0][pages][..., None])


def value_values(state, pages):
    """Values of pages [...], [..., kv_heads, 128, 16]."""
    codes = state["codes"][:, :, 1][pages].unflatten(-1, (HEAD, PAGE))
    return values(codes, state["scales"][:, :, 1][pages][..., None, :])


def cache(case, seed, g):
    """Pages in shuffled order, every one filled: keys of unit size with a few strong dims that drift along the
    sequence, values around 1; and the bounds of the keys."""
    kvh, n, per = case["kv_heads"], case["seqs"], pages_of(case)
    pool = n * per + 3
    table = torch.randperm(pool, device="cuda", generator=g)[:n * per].to(torch.int32).view(n, per)
    drift = normal(g, (pool, kvh, 1, HEAD)) * (torch.rand((1, kvh, 1, HEAD), device="cuda", generator=g) < 0.1) * 3.0
    k = (normal(g, (pool, kvh, PAGE, HEAD)) + drift).bfloat16().float()
    kc, ks = quantise(k)
    v = normal(g, (pool, kvh, PAGE, HEAD)).bfloat16().float()
    vc, vs = quantise(v)
    held = values(kc, ks[..., None])
    return {"case": case, "table": table, "pool": pool,
            "codes": torch.stack([kc.flatten(-2), vc.transpose(-1, -2).flatten(-2)], 2),
            "scales": torch.stack([ks, vs], 2).contiguous(),
            "bounds": torch.stack([held.amin(-2), held.amax(-2)], 2).bfloat16()}


def prepare(case, seed):
    g = generator(seed)
    state = cache(case, seed, g)
    if case["op"] == "write":
        qh, kvh, rows = case["q_heads"], case["kv_heads"], case["rows"]
        seq, pos = write_rows(case, seed)
        inv = (1.0 / THETA ** (torch.arange(0, HEAD, 2, dtype=torch.float64, device="cuda") / HEAD)).float()
        angle = (torch.arange(case["longest"], dtype=torch.float32, device="cuda")[:, None] * inv).double()
        state |= {"qkv": (normal(g, (rows, qh + 2 * kvh, HEAD)) * 2.0).bfloat16(),
                  "q_norm": (1.0 + 0.2 * normal(g, (HEAD,))).bfloat16(),
                  "k_norm": (1.0 + 0.2 * normal(g, (HEAD,))).bfloat16(),
                  "rope": torch.stack([torch.cos(angle), torch.sin(angle)], -1).contiguous(),
                  "row_seq": torch.from_numpy(seq.astype(np.int32)).cuda(),
                  "row_pos": torch.from_numpy(pos.astype(np.int32)).cuda(),
                  "q_out": torch.zeros((rows, qh, HEAD), dtype=torch.bfloat16, device="cuda")}
        return state
    state["lens"] = torch.from_numpy(host(seed).permutation(lengths(case)).astype(np.int32)).cuda()
    if case["op"] == "read":
        n, per, kvh = case["seqs"], pages_of(case), case["kv_heads"]
        shape = (n * per, kvh, PAGE, HEAD)
        state |= {"out_table": torch.randperm(n * per, device="cuda", generator=g).to(torch.int32).view(n, per),
                  "k": torch.zeros(shape, dtype=torch.bfloat16, device="cuda"),
                  "v": torch.zeros((n * per, kvh, HEAD, PAGE), dtype=torch.bfloat16, device="cuda")}
        return state
    shape = (case["seqs"], case["q_heads"], HEAD)
    state |= {"q": (normal(g, shape) * 1.5).bfloat16(), "out": torch.zeros(shape, dtype=torch.bfloat16, device="cuda")}
    if case["op"] == "sparse":
        state["list"] = torch.zeros((case["seqs"], case["kv_heads"], case["budget"]), dtype=torch.int32, device="cuda")
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


def workspace(size):
    """The program's one workspace, zeroed once."""
    if "work" not in _kept or _kept["work"].numel() < size:
        gpu().sync()
        _kept["work"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return _kept["work"].data_ptr(), _kept["work"].numel()


def run_own(state):
    g, case = gpu(), state["case"]
    from x0ne_core import Kv8
    at = {k: v.data_ptr() for k, v in state.items() if isinstance(v, torch.Tensor)}
    kv = Kv8(codes=at["codes"], scales=at["scales"], page_table=at["table"], pool=state["pool"], kv_heads=case["kv_heads"],
             seqs=case["seqs"], seq_pages=pages_of(case))
    if case["op"] == "write":
        g.kv8_write(kv, at["qkv"], case["rows"], case["q_heads"], at["q_norm"], at["k_norm"], EPS, at["rope"], case["longest"],
                    at["row_seq"], at["row_pos"], at["q_out"], bounds=at["bounds"])
    elif case["op"] == "read":
        g.kv8_read(kv, at["lens"], at["k"], at["v"], at["out_table"], state["k"].shape[0])
    else:
        work = workspace(g.kv8_work_bytes(kv, case["q_heads"]))
        if case["op"] == "sparse":
            g.kv8_select(kv, at["bounds"], at["q"], case["q_heads"], at["lens"], case["budget"], at["list"], *work)
            g.kv8_attention(kv, at["q"], case["q_heads"], at["lens"], at["out"], SCALE, *work, page_list=at["list"],
                            budget=case["budget"])
        else:
            g.kv8_attention(kv, at["q"], case["q_heads"], at["lens"], at["out"], SCALE, *work)


# -- the plain form --

def rope_norm(x, w, cos, sin):
    """The RMSNorm of each head, rotated, in 64 bits: the rounding to bf16 decides the codes."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    a, b = x[..., :HALF], x[..., HALF:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float().bfloat16()


def plain_write(state):
    case = state["case"]
    qh, kvh = case["q_heads"], case["kv_heads"]
    live = state["row_seq"] >= 0
    seq, pos = state["row_seq"].clamp(min=0).long(), state["row_pos"].long()
    cos, sin = state["rope"][pos, :, 0][:, None], state["rope"][pos, :, 1][:, None]
    q = rope_norm(state["qkv"][:, :qh], state["q_norm"], cos, sin)
    k = rope_norm(state["qkv"][:, qh:qh + kvh], state["k_norm"], cos, sin)
    state["q_out"].copy_(torch.where(live[:, None, None], q, state["q_out"]))
    page, slot = state["table"][seq, pos // PAGE].long()[live], (pos % PAGE)[live]
    kc, ks = quantise(k[live].float())
    vc, vs = quantise(state["qkv"][:, qh + kvh:][live].float())
    keys = state["codes"][:, :, 0].unflatten(-1, (PAGE, HEAD))
    vals = state["codes"][:, :, 1].unflatten(-1, (HEAD, PAGE))
    keys[page, :, slot] = kc
    vals[page, :, :, slot] = vc
    state["scales"][page, :, 0, slot] = ks
    state["scales"][page, :, 1, slot] = vs
    whole = page[slot == PAGE - 1]
    held = key_values(state, whole)
    state["bounds"][whole] = torch.stack([held.amin(-2), held.amax(-2)], 2).bfloat16()


def gathered(state):
    """Keys and values in 32 bits, [seqs][kv_heads][positions][128] both, zero past a sequence's length, and which
    positions a sequence has."""
    case = state["case"]
    t = state["table"].long()
    k, v = key_values(state, t), value_values(state, t).transpose(-1, -2)
    k, v = (x.permute(0, 2, 1, 3, 4).reshape(case["seqs"], case["kv_heads"], -1, HEAD) for x in (k, v))
    here = torch.arange(k.shape[2], device="cuda")[None] < state["lens"][:, None]
    return k.masked_fill(~here[:, None, :, None], 0.0), v.masked_fill(~here[:, None, :, None], 0.0), here


def plain_read(state):
    case = state["case"]
    n, per, kvh = case["seqs"], pages_of(case), case["kv_heads"]
    k, v, _ = gathered(state)
    k, v = (x.view(n, kvh, per, PAGE, HEAD).transpose(1, 2).bfloat16() for x in (k, v))
    used = torch.arange(per, device="cuda")[None] * PAGE < state["lens"][:, None]
    at = state["out_table"].long()[used]
    state["k"][at] = k[used]
    state["v"][at] = v[used].transpose(-1, -2)


def attend(q, k, v, keep):
    """Softmax attention in 32 bits over the keys that keep [seqs][kv_heads][positions] allows."""
    n, qh, kvh = q.shape[0], q.shape[1], k.shape[1]
    s = q.float().view(n, kvh, qh // kvh, HEAD) @ k.transpose(-1, -2) * SCALE
    s = s.masked_fill(~keep[:, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return ((p @ v) / torch.where(total > 0, total, 1.0)).reshape(n, qh, HEAD).bfloat16()


def plain_attend(state):
    k, v, here = gathered(state)
    state["out"].copy_(attend(state["q"], k, v, here[:, None].expand(-1, k.shape[1], -1)))


def chosen(state):
    """The pages of each sequence and kv head, in 64 bits: a page next to the border decides what is read."""
    case = state["case"]
    n, kvh, per, budget = case["seqs"], case["kv_heads"], pages_of(case), case["budget"]
    q = state["q"].double().view(n, kvh, -1, HEAD)
    b = state["bounds"][state["table"].long()].double().permute(3, 0, 2, 4, 1)  # [2][seqs][kv_heads][128][pages]
    score = (q.clamp(min=0.0) @ b[1].contiguous() + q.clamp(max=0.0) @ b[0].contiguous()).amax(2)
    count = (state["lens"].long() + PAGE - 1) // PAGE
    page = torch.arange(per, device="cuda")
    score = torch.where(page == count[:, None, None] - 1, math.inf, score)
    score = torch.where(page >= count[:, None, None], -math.inf, score)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    best = torch.where(best < count[:, None, None], best, per).sort(-1).values
    best = torch.cat([best, best.new_full((n, kvh, max(0, budget - per)), per)], -1)
    return torch.where(best < per, best, -1)


def plain_sparse(state):
    ids = chosen(state)
    state["list"].copy_(ids)
    k, v, here = gathered(state)
    n, kvh, per = k.shape[0], k.shape[1], pages_of(state["case"])
    keep = torch.zeros((n, kvh, per + 1), dtype=torch.bool, device="cuda").scatter_(-1, torch.where(ids < 0, per, ids), True)
    keep = keep[..., :per].repeat_interleave(PAGE, -1) & here[:, None]
    state["out"].copy_(attend(state["q"], k, v, keep))


def run(state):
    op = state["case"]["op"]
    if own:
        run_own(state)
    else:
        {"write": plain_write, "read": plain_read, "attend": plain_attend, "sparse": plain_sparse}[op](state)
    if op == "write":
        return {"q": state["q_out"], "codes": state["codes"].view(torch.float8_e4m3fn), "scales": state["scales"],
                "bounds": state["bounds"]}
    if op == "read":
        return {"k": state["k"], "v": state["v"]}
    return {"out": state["out"], "list": state["list"]} if op == "sparse" else {"out": state["out"]}


# -- what a pass cannot do without --

def work(case):
    kvh = case["kv_heads"]
    row = kvh * 2 * (HEAD + 1)  # a position's codes and scale bytes
    if case["op"] == "write":
        rows, qh = case["rows"], case["q_heads"]
        return {"bytes": rows * (2 * HEAD * (2 * qh + 2 * kvh) + row + 16 * HALF + 8) + 4 * HEAD, "flops": rows * (qh + kvh) * HEAD * 8}
    lens = lengths(case)
    keys, pages = int(lens.sum()), int((-(-lens // PAGE)).sum())
    if case["op"] == "read":
        return {"bytes": keys * (row + kvh * 4 * HEAD), "flops": 0}
    qo = case["seqs"] * case["q_heads"] * HEAD * 4
    if case["op"] == "attend":
        return {"bytes": keys * row + qo, "flops": keys * case["q_heads"] * HEAD * 4}
    keys = int(np.minimum(lens, case["budget"] * PAGE).sum())
    return {"bytes": keys * row + pages * kvh * 4 * HEAD + qo, "flops": case["q_heads"] * HEAD * 4 * (keys + pages)}


# -- the same in 64 bits, row by row from the definition --

def e4m3_grid():
    """The 127 magnitudes of e4m3, by code."""
    c = np.arange(127)
    return np.where(c < 8, c * 2.0 ** -9, (1.0 + c % 8 / 8.0) * 2.0 ** (c // 8 - 7.0))


def nearest_code(x):
    """e4m3 codes of f64 values of at most 448: the nearest magnitude, the even code where two are as near."""
    grid = e4m3_grid()
    a = np.abs(x)
    hi = np.searchsorted(grid, a).clip(1, 126)
    lo = hi - 1
    up = (grid[hi] - a < a - grid[lo]) | ((grid[hi] - a == a - grid[lo]) & (hi % 2 == 0))
    return np.where(up, hi, lo) + np.where(np.signbit(x), 128, 0)


def bf16_of(x):
    """f64 values rounded to bf16 through f32, as f64."""
    return torch.from_numpy(x).float().bfloat16().double().numpy()


def exact_rows(x, w, cos, sin):
    x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + EPS) * w
    turned = (x[..., :HALF] + 1j * x[..., HALF:]) * (cos + 1j * sin)[:, None]
    return np.concatenate([turned.real, turned.imag], -1)


def exact_quantise(x):
    top = np.abs(x).max(-1)
    with np.errstate(divide="ignore"):
        e = np.maximum(np.ceil(np.log2(top / 448.0)), LOWEST)
    e = np.where(top > 448.0 * 2.0 ** e, e + 1, e)
    e = np.maximum(np.where((top <= 448.0 * 2.0 ** (e - 1)), e - 1, e), LOWEST)
    return nearest_code(x / 2.0 ** e[..., None]), e.astype(np.int64) + 127


def numbers(t):
    return t.cpu().double().numpy()


def exact_write(s, case):
    qh, kvh = case["q_heads"], case["kv_heads"]
    x, seq, pos = numbers(s["qkv"]), s["row_seq"].cpu().numpy(), s["row_pos"].cpu().numpy()
    live, rope = np.nonzero(seq >= 0)[0], s["rope"].cpu().numpy()[pos]
    q = exact_rows(x[:, :qh], numbers(s["q_norm"]), rope[..., 0], rope[..., 1])
    k = exact_rows(x[:, qh:qh + kvh], numbers(s["k_norm"]), rope[..., 0], rope[..., 1])
    q_out = np.zeros_like(q)
    q_out[live] = q[live]
    kc, ke = exact_quantise(bf16_of(k[live]))
    vc, ve = exact_quantise(x[live, qh + kvh:])
    codes, scales, bounds = s["codes"].cpu().numpy().copy(), s["scales"].cpu().numpy().copy(), numbers(s["bounds"])
    table, grid = s["table"].cpu().numpy(), np.concatenate([e4m3_grid(), [np.nan], -e4m3_grid(), [np.nan]])
    for i, r in enumerate(live):
        page, slot = table[seq[r], pos[r] // PAGE], pos[r] % PAGE
        codes[page, :, 0, slot * HEAD:(slot + 1) * HEAD] = kc[i]
        codes[page, :, 1, slot::PAGE] = vc[i]
        scales[page, :, 0, slot], scales[page, :, 1, slot] = ke[i], ve[i]
    for r in live[pos[live] % PAGE == PAGE - 1]:
        page = table[seq[r], pos[r] // PAGE]
        held = grid[codes[page, :, 0]].reshape(kvh, PAGE, HEAD) * 2.0 ** (scales[page, :, 0].astype(np.float64) - 127)[..., None]
        bounds[page] = np.stack([held.min(1), held.max(1)], 1)
    return {"q": q_out, "codes": grid[codes], "scales": scales, "bounds": bounds}


def exact_sequence(s, i, per, kvh):
    """Keys and values of sequence i in 64 bits, [kv_heads][its length][128], on the GPU."""
    n = int(s["lens"][i])
    at = s["table"][i, :-(-n // PAGE)].long()
    power = torch.pow(2.0, s["scales"][at].double() - 127.0)
    grid = torch.from_numpy(np.concatenate([e4m3_grid(), [np.nan], -e4m3_grid(), [np.nan]])).cuda()
    c = grid[s["codes"][at].long()]
    k = c[:, :, 0].reshape(-1, kvh, PAGE, HEAD) * power[:, :, 0, :, None]
    v = c[:, :, 1].reshape(-1, kvh, HEAD, PAGE) * power[:, :, 1, None, :]
    return (k.permute(1, 0, 2, 3).reshape(kvh, -1, HEAD)[:, :n], v.permute(1, 0, 3, 2).reshape(kvh, -1, HEAD)[:, :n])


def exact_read(s, case):
    kvh = case["kv_heads"]
    out_k, out_v = torch.zeros_like(s["k"], dtype=torch.float64), torch.zeros_like(s["v"], dtype=torch.float64)
    for i in range(case["seqs"]):
        k, v = exact_sequence(s, i, pages_of(case), kvh)
        for p in range(-(-k.shape[1] // PAGE)):
            at, m = int(s["out_table"][i, p]), min(PAGE, k.shape[1] - p * PAGE)
            out_k[at, :, :m] = k[:, p * PAGE:p * PAGE + m]
            out_v[at, :, :, :m] = v[:, p * PAGE:p * PAGE + m].transpose(1, 2)
    return {"k": out_k, "v": out_v}


def exact_pages(s, case, i, q):
    """The pages that sequence i reads for kv head h, ascending."""
    kvh, n = case["kv_heads"], int(s["lens"][i])
    count = -(-n // PAGE)
    if count == 0:
        return [np.array([], np.int64)] * kvh
    b = numbers(s["bounds"][s["table"][i, :count].long()])  # [pages][kv_heads][2][128]
    picked = []
    for h in range(kvh):
        qs = q.reshape(kvh, -1, 1, HEAD)[h]
        score = np.maximum(qs * b[:, h, 0], qs * b[:, h, 1]).sum(-1).max(0)[:-1]
        order = np.lexsort((np.arange(count - 1), -score))[:case["budget"] - 1]
        picked.append(np.sort(np.append(order, count - 1)))
    return picked


def exact_attention(s, case):
    kvh, sparse = case["kv_heads"], case["op"] == "sparse"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    ids = np.full((case["seqs"], kvh, case.get("budget", 0)), -1)
    for i in range(case["seqs"]):
        k, v = exact_sequence(s, i, pages_of(case), kvh)
        n = k.shape[1]
        if n == 0:
            continue
        logits = torch.bmm(s["q"][i].double().view(kvh, -1, HEAD), k.transpose(1, 2).contiguous()) / math.sqrt(HEAD)
        if sparse:
            keep = torch.zeros((kvh, n), dtype=torch.bool)
            for h, pages in enumerate(exact_pages(s, case, i, numbers(s["q"][i]))):
                ids[i, h, :len(pages)] = pages
                at = (pages[:, None] * PAGE + np.arange(PAGE)).reshape(-1)
                keep[h, torch.from_numpy(at[at < n])] = True
            logits = logits.masked_fill(~keep.cuda()[:, None], -math.inf)
        out[i] = torch.bmm(torch.softmax(logits, -1), v.contiguous()).reshape(-1, HEAD)
    return {"out": out, "list": torch.from_numpy(ids)} if sparse else {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": exact_write, "read": exact_read, "attend": exact_attention, "sparse": exact_attention}[case["op"]](s, case)
