"""Workloads of the ragged-batch operators: request plan, gated delta rule, 8-bit matrix product.

Four operators that a serving step over a pool of recurrent-state slots uses together:

  plan    token offsets, state slots, per-token maps and the block table of a ragged batch, from
          the requests' lengths (PluginLibrary.plan_requests)
  chunk   the gated delta rule over whole windows, each request from its slot's state
          (PluginLibrary.delta_chunk)
  step    the same rule for one token of each stream (PluginLibrary.delta_step)
  linear  x -> per-token int8 -> product with per-channel int8 weights
          (PluginLibrary.w8a8_linear); with x "int8" the product alone (PluginLibrary.w8a8_matmul)

`run` computes an operator in plain 32-bit torch operations, or through the framework's entry
points when `own` is set; `exact` computes it from its definition in 64 bits.

The rule, per value head (S is dv x dk, q and k are divided by their 2-norms where `l2norm`):
    S_t = a_t S_{t-1} + b_t (v_t - a_t S_{t-1} k_t) k_t^T,   a_t = exp(g_t),   o_t = scale S_t q_t
"""
import math
import random

import numpy as np
import torch

own = False

NONE = -1           # a request without a slot (the entry points' UINT32_MAX)
EPS = 1e-6          # of the 2-norm: x / sqrt(sum x^2 + EPS)
CHUNK = 64          # tokens per step of the plain chunked form
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"f32": 0, "bf16": 1}
_library = None


def library():
    global _library
    if _library is None:
        from redukt_b200.plugin import PluginLibrary
        _library = PluginLibrary()
    return _library


# ---- cases -----------------------------------------------------------------------------------

def listed():
    return [
        # a decode step's admission: a handful of new windows join a pool of 32 lockstep streams
        {"name": "plan_small", "op": "plan", "n": 8, "mean": 40, "slots": 32, "block": 64},
        # the whole pool of 4,096 slots is planned for a prefill of about two million tokens
        {"name": "plan_pool", "op": "plan", "n": 4096, "mean": 512, "slots": 4096, "block": 256},
        # one lockstep step: 32 streams, 12 heads of 64, everything f32
        {"name": "step_lockstep", "op": "step", "n": 32, "hk": 12, "hv": 12, "dk": 64, "dv": 64, "dtype": "f32",
         "l2norm": True},
        # a step of a large pool with grouped heads: the state (268 MB) is what moves
        {"name": "step_pool", "op": "step", "n": 256, "hk": 8, "hv": 16, "dk": 128, "dv": 128, "dtype": "bf16",
         "l2norm": True},
        # three prompts of a few tokens: only latency counts
        {"name": "chunk_short", "op": "chunk", "n": 3, "mean": 8, "spread": 3.0, "hk": 12, "hv": 12, "dk": 64, "dv": 64,
         "dtype": "bf16", "l2norm": True},
        # 32 equal windows of 2,700 tokens, 12 heads of 64, f32
        {"name": "chunk_windows_f32", "op": "chunk", "n": 32, "mean": 2700, "spread": 0.0, "hk": 12, "hv": 12, "dk": 64,
         "dv": 64, "dtype": "f32", "l2norm": True},
        # a ragged prefill with empty requests, grouped heads of 128; keys are normalised by the caller
        {"name": "chunk_ragged", "op": "chunk", "n": 64, "mean": 350, "spread": 2.5, "hk": 8, "hv": 16, "dk": 128,
         "dv": 128, "dtype": "bf16", "l2norm": False},
        # one long document alone on the GPU: few chains, many chunks
        {"name": "chunk_long", "op": "chunk", "n": 1, "mean": 16384, "spread": 0.0, "hk": 4, "hv": 8, "dk": 128, "dv": 128,
         "dtype": "bf16", "l2norm": True},
        # the logits of one stream: a 65,536 x 768 head on one token
        {"name": "linear_head", "op": "linear", "m": 1, "n": 65536, "k": 768, "x": "f32", "out": "f32"},
        # a fused q/k/v projection of 32 lockstep streams
        {"name": "linear_lockstep", "op": "linear", "m": 32, "n": 2304, "k": 768, "x": "f32", "out": "f32"},
        # a prefill's projection: enough rows to fill the tensor cores
        {"name": "linear_prefill", "op": "linear", "m": 16384, "n": 8192, "k": 4096, "x": "bf16", "out": "bf16"},
        # odd sizes, quantised inputs in hand
        {"name": "matmul_odd", "op": "linear", "m": 777, "n": 1111, "k": 1000, "x": "int8", "out": "f32"},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "step", "chunk", "chunk", "linear", "linear"])
    if op == "plan":
        n = log_int(rng, 1, 4096)
        return {"op": op, "n": n, "mean": log_int(rng, 1, 512), "slots": log_int(rng, 16, 4096),
                "block": rng.choice([64, 128, 256, 1024])}
    if op == "linear":
        x = rng.choice(["f32", "bf16", "bf16", "int8"])
        while True:
            m, n, k = log_int(rng, 1, 16384), log_int(rng, 64, 65536), log_int(rng, 64, 8192)
            if n != 3072 and k != 3072 and m * n * k <= 5e11 and 4 * m * n + n * k <= 2e9:
                return {"op": op, "m": m, "n": n, "k": k, "x": x, "out": rng.choice(["f32", "bf16"])}
    group = rng.choice([1, 1, 2, 4])
    hk = log_int(rng, 1, 16)
    case = {"op": op, "hk": hk, "hv": hk * group, "dk": rng.choice([64, 128]), "dv": rng.choice([64, 128]),
            "dtype": rng.choice(["f32", "bf16"]), "l2norm": rng.random() < 0.7}
    per = case["hv"] * case["dk"] * case["dv"]
    while True:
        if op == "step":
            case["n"] = log_int(rng, 1, 512)
            if case["n"] * per <= 6.5e7:
                return case
        else:
            case.update(n=log_int(rng, 1, 64), mean=log_int(rng, 2, 8192), spread=rng.choice([0.0, 1.5, 3.0]))
            total = case["n"] * case["mean"]
            if total <= 60000 and total * per <= 4.5e9:
                return case


def lengths_of(case):
    """Request lengths: a property of the case (the byte count depends on them), not of the seed."""
    r = random.Random(1000003 * case["n"] + case["mean"])
    if case["op"] == "plan":  # geometric-like, one in sixteen empty
        return [0 if r.random() < 1 / 16 else 1 + int(r.expovariate(1.0 / case["mean"])) for _ in range(case["n"])]
    if not case["spread"]:
        return [case["mean"]] * case["n"]
    cap = int(case["spread"] * case["mean"])
    got = [0 if r.random() < 1 / 16 else r.randint(1, max(1, min(cap, 2 * case["mean"] - 1))) for _ in range(case["n"])]
    got[r.randrange(case["n"])] = cap  # one request much longer than the others
    return got


def work(case):
    op = case["op"]
    if op == "plan":
        n, total, block = case["n"], sum(lengths_of(case)), case["block"]
        blocks = total // block + n
        return {"bytes": 4 * 2 * n + 2 * case["slots"] + 4 * (2 * (n + 1) + 2 * n) + 8 * total + 8 * blocks, "flops": 0}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = {"f32": 4 * m * k, "bf16": 2 * m * k, "int8": m * k + 4 * m}[case["x"]]
        return {"bytes": x + n * k + 4 * n + m * n * (4 if case["out"] == "f32" else 2), "flops": 2 * m * n * k}
    size = 4 if case["dtype"] == "f32" else 2
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    rows = case["n"] if op == "step" else sum(lengths_of(case))
    states = case["n"]
    return {"bytes": rows * (size * (2 * hk * dk + 2 * hv * dv) + 8 * hv) + 2 * 4 * states * hv * dv * dk,
            "flops": 6 * rows * hv * dv * dk}


# ---- inputs ----------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = "cuda"

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    if case["op"] == "plan":
        n, slots = case["n"], case["slots"]
        lens = torch.tensor(lengths_of(case), dtype=torch.int32, device=dev)
        # the lengths in another order for each seed; about half of the slots are in use, and one
        # request in four continues a stream (now and then two ask for the same one)
        lens = lens[torch.randperm(n, generator=gen, device=dev)].contiguous()
        used = (uniform(slots) < 0.5).to(torch.uint8)
        want = torch.randint(0, slots, (n,), generator=gen, device=dev, dtype=torch.int32)
        want = torch.where(uniform(n) < 0.25, want, torch.full_like(want, NONE))
        tokens = sum(lengths_of(case))
        blocks = tokens // case["block"] + n

        def out(*shape, dtype=torch.int32):
            return torch.empty(*shape, dtype=dtype, device=dev)

        return {"case": case, "lens": lens, "want": want, "used": used, "max_tokens": tokens, "max_blocks": blocks,
                "cu": out(n + 1), "slot": out(n), "fresh": out(n), "used_out": out(slots, dtype=torch.uint8),
                "token_slot": out(tokens), "token_pos": out(tokens), "block_base": out(n + 1), "blocks": out(blocks, 2)}

    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        ld = (k + 15) // 16 * 16  # int8 rows start on 16 bytes
        w = torch.zeros(n, ld, dtype=torch.int8, device=dev)
        w[:, :k] = torch.clamp(torch.round(normal(n, k) * 32), -127, 127).to(torch.int8)
        w_scale = (0.5 + uniform(n)) * (0.02 / 32)
        s = {"case": case, "w": w, "w_scale": w_scale, "out": torch.empty(m, n, dtype=DTYPES[case["out"]], device=dev)}
        if case["x"] == "int8":
            x = torch.zeros(m, ld, dtype=torch.int8, device=dev)
            x[:, :k] = torch.clamp(torch.round(normal(m, k) * 32), -127, 127).to(torch.int8)
            s.update(x=x, x_scale=(0.5 + uniform(m)) / 32)
        else:
            # activations with a few channels much larger than the rest
            x = normal(m, k) * torch.where(uniform(k) < 0.01, 10.0, 1.0)
            s["x"] = x.to(DTYPES[case["x"]])
        s["work"] = torch.empty(m * ld + 4 * m + (1 << 26), dtype=torch.uint8, device=dev)
        return s

    n, hk, hv, dk, dv = case["n"], case["hk"], case["hv"], case["dk"], case["dv"]
    t = DTYPES[case["dtype"]]
    lens = [1] * n if case["op"] == "step" else lengths_of(case)
    rows, slots = sum(lens), n + 1
    q, k, v = normal(rows, hk, dk), normal(rows, hk, dk), normal(rows, hv, dv)
    if not case["l2norm"]:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
    # decay rates 1..16 per head, step sizes log-uniform in [1e-3, 1e-1]
    rate = 1.0 + 15.0 * uniform(hv)
    g = -rate * torch.exp(math.log(1e-3) + uniform(rows, hv) * math.log(100.0))
    s = {"case": case, "lens": lens, "q": q.to(t), "k": k.to(t), "v": v.to(t), "g": g.contiguous(),
         "beta": torch.sigmoid(normal(rows, hv)), "scale": 1.0 / math.sqrt(dk),
         "state": 0.3 * normal(slots, hv, dv, dk),
         "slot": torch.randperm(slots, generator=gen, device=dev)[:n].to(torch.int32),
         "fresh": (uniform(n) < 0.5).to(torch.int32), "out": torch.empty(rows, hv, dv, dtype=t, device=dev)}
    if case["op"] == "chunk":  # the plan of the batch, as plan_requests gives it
        block = 256
        cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        table = [(i, j) for i, size in enumerate(lens) for j in range((size + block - 1) // block)]
        most = rows // block + n
        table += [(NONE, NONE)] * (most - len(table))
        s.update(cu=torch.from_numpy(cu).to(dev), block=block, max_blocks=most,
                 blocks=torch.tensor(table, dtype=torch.int32, device=dev).reshape(most, 2))
        s["work"] = torch.empty(1 << 29, dtype=torch.uint8, device=dev)
    return s


# ---- one pass --------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"plan": own_plan, "linear": own_linear, "chunk": own_chunk, "step": own_step}[op](s)
    return {"plan": plain_plan, "linear": plain_linear, "chunk": plain_chunk, "step": plain_step}[op](s)


def plan_outputs(s):
    return {k: s[k] for k in ("cu", "slot", "fresh", "used_out", "token_slot", "token_pos", "block_base", "blocks")}


def checked(code):
    if code != 0:
        raise RuntimeError("%s: %s" % (code.name, library().last_error()))


def own_plan(s):
    c = s["case"]
    checked(library().plan_requests(
        s["lens"].data_ptr(), s["want"].data_ptr(), c["n"], s["used"].data_ptr(), c["slots"], c["block"],
        s["max_tokens"], s["max_blocks"], s["cu"].data_ptr(), s["slot"].data_ptr(), s["fresh"].data_ptr(),
        s["used_out"].data_ptr(), s["token_slot"].data_ptr(), s["token_pos"].data_ptr(), s["block_base"].data_ptr(),
        s["blocks"].data_ptr(), torch.cuda.current_stream().cuda_stream))
    return plan_outputs(s)


def own_linear(s):
    c, x, w = s["case"], s["x"], s["w"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["x"] == "int8":
        checked(library().w8a8_matmul(
            x.data_ptr(), x.stride(0), s["x_scale"].data_ptr(), c["m"], w.data_ptr(), w.stride(0), s["w_scale"].data_ptr(),
            c["n"], c["k"], s["out"].data_ptr(), CODES[c["out"]], c["n"], s["work"].data_ptr(), s["work"].numel(), stream))
    else:
        checked(library().w8a8_linear(
            x.data_ptr(), CODES[c["x"]], c["m"], c["k"], x.stride(0), w.data_ptr(), w.stride(0), s["w_scale"].data_ptr(),
            c["n"], s["out"].data_ptr(), CODES[c["out"]], c["n"], s["work"].data_ptr(), s["work"].numel(), stream))
    return s["out"]


def own_step(s):
    c = s["case"]
    checked(library().delta_step(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), CODES[c["dtype"]], s["g"].data_ptr(), s["beta"].data_ptr(),
        c["n"], s["slot"].data_ptr(), s["fresh"].data_ptr(), c["hk"], c["hv"], c["dk"], c["dv"],
        s["q"].stride(0), s["k"].stride(0), s["v"].stride(0), s["g"].stride(0), s["out"].stride(0),
        s["scale"], int(c["l2norm"]), s["state"].data_ptr(), s["state"].shape[0], s["state"].stride(0),
        s["out"].data_ptr(), torch.cuda.current_stream().cuda_stream))
    return {"out": s["out"], "state": s["state"]}


def own_chunk(s):
    c = s["case"]
    checked(library().delta_chunk(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), CODES[c["dtype"]], s["g"].data_ptr(), s["beta"].data_ptr(),
        s["q"].shape[0], c["n"], s["cu"].data_ptr(), s["slot"].data_ptr(), s["fresh"].data_ptr(),
        c["hk"], c["hv"], c["dk"], c["dv"],
        s["q"].stride(0), s["k"].stride(0), s["v"].stride(0), s["g"].stride(0), s["out"].stride(0),
        s["scale"], int(c["l2norm"]), s["state"].data_ptr(), s["state"].shape[0], s["state"].stride(0),
        s["blocks"].data_ptr(), s["block"], s["max_blocks"], s["out"].data_ptr(), s["work"].data_ptr(),
        s["work"].numel(), torch.cuda.current_stream().cuda_stream))
    return {"out": s["out"], "state": s["state"]}


def plain_plan(s):
    c = s["case"]
    n, slots, block, most = c["n"], c["slots"], c["block"], s["max_tokens"]
    lens, want, used = s["lens"].long(), s["want"].long(), s["used"] != 0
    dev = lens.device
    end = torch.cumsum(lens, 0)
    cu = torch.cat([end.new_zeros(1), end.clamp(max=most)])
    live = (lens > 0) & (end <= most)
    # a slot that two requests ask for goes to the first of them
    named = (want >= 0) & (want < slots)
    at = torch.where(named, want, torch.full_like(want, slots))
    index = torch.arange(n, device=dev)
    owner = torch.full((slots + 1,), n, dtype=torch.long, device=dev).scatter_reduce(0, at, index, "amin")
    keeps = named & (owner[at] == index) & (end <= most)
    taken = used | (owner[:slots] < n)
    # the lowest free slots go to the new requests in their order
    free = torch.nonzero(~taken).flatten()
    new = live & (want == NONE)
    rank = torch.cumsum(new.long(), 0) - 1
    admitted = new & (rank < free.numel())
    padded = torch.cat([free, free.new_full((1,), NONE)])
    slot = torch.where(keeps, want, torch.where(admitted, padded[rank.clamp(0, free.numel())], torch.full_like(want, NONE)))
    used_out = taken.clone()
    used_out[slot[admitted]] = True
    t = torch.arange(most, device=dev)
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=n - 1)
    inside = t < cu[n]
    token_slot = torch.where(inside, slot[req], torch.full_like(t, NONE))
    token_pos = torch.where(inside, t - cu[req], torch.full_like(t, NONE))
    count = (cu[1:] - cu[:-1] + block - 1) // block
    base = torch.cat([count.new_zeros(1), torch.cumsum(count, 0)])
    b = torch.arange(s["max_blocks"], device=dev)
    breq = torch.searchsorted(base[1:].contiguous(), b, right=True).clamp(max=n - 1)
    bin_ = (b < base[n])[:, None]
    blocks = torch.where(bin_, torch.stack([breq, b - base[breq]], 1), torch.full((1, 2), NONE, device=dev))
    got = {"cu": cu, "slot": slot, "fresh": admitted, "token_slot": token_slot, "token_pos": token_pos,
           "block_base": base, "blocks": blocks}
    return {**{k: v.to(torch.int32) for k, v in got.items()}, "used_out": used_out.to(torch.uint8)}


def plain_linear(s):
    c, k = s["case"], s["case"]["k"]
    w = s["w"][:, :k].float()
    if c["x"] == "int8":
        x, scale = s["x"][:, :k].float(), s["x_scale"]
    else:
        x = s["x"].float()
        amax = x.abs().amax(1)
        scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
        t = x * (1.0 / scale)[:, None]
        # round half away from zero: t - trunc(t) is exact
        whole = torch.trunc(t)
        x = (whole + torch.sign(t) * ((t - whole).abs() >= 0.5)).clamp(-127, 127)
    return ((x @ w.T) * (s["w_scale"][None, :] * scale[:, None])).to(DTYPES[c["out"]])


def plain_heads(s):
    """q, k, v as 32-bit [rows, hv, d], normalised where asked, each q/k head repeated for its group."""
    c = s["case"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["l2norm"]:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
    group = c["hv"] // c["hk"]
    return q.repeat_interleave(group, 1), k.repeat_interleave(group, 1), v


def start_states(s):
    return s["state"][s["slot"].long()] * (s["fresh"] == 0).float()[:, None, None, None]


def plain_step(s):
    q, k, v = plain_heads(s)
    S = start_states(s) * torch.exp(s["g"])[:, :, None, None]
    u = s["beta"][:, :, None] * (v - (S * k[:, :, None, :]).sum(-1))
    S = S + u[:, :, :, None] * k[:, :, None, :]
    s["out"].copy_(s["scale"] * (S * q[:, :, None, :]).sum(-1))
    s["state"][s["slot"].long()] = S
    return {"out": s["out"], "state": s["state"]}


def unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a [..., 64, 64], by halves: 1, 2, 4, ... 32."""
    x = torch.eye(CHUNK, device=a.device).expand_as(a).clone()
    lead = a.shape[:-2]
    size = 1
    while size < CHUNK:
        m = CHUNK // (2 * size)
        pair = torch.arange(m, device=a.device)
        xb, ab = (y.reshape(*lead, m, 2, size, m, 2, size) for y in (x, a))
        upper = xb[..., pair, 0, :, pair, 0, :]  # [m, ..., size, size]
        lower = xb[..., pair, 1, :, pair, 1, :]
        cross = ab[..., pair, 1, :, pair, 0, :]
        xb[..., pair, 1, :, pair, 0, :] = -(lower @ (cross @ upper))
        size *= 2
    return x


def plain_chunk(s):
    c = s["case"]
    n, hv, dk, dv, lens = c["n"], c["hv"], c["dk"], c["dv"], s["lens"]
    dev = s["q"].device
    q, k, v = plain_heads(s)
    chunks = (max(lens) + CHUNK - 1) // CHUNK
    # every request padded to `chunks` chunks; a padded token has k = v = 0, g = 0, beta = 0
    t = torch.arange(chunks * CHUNK, device=dev)
    size = torch.tensor(lens, device=dev)
    inside = t[None, :] < size[:, None]
    row = torch.where(inside, s["cu"][:-1].long()[:, None] + t[None, :], torch.full((1, 1), q.shape[0], device=dev))

    def laid(x, *tail):  # [n, chunks, hv, CHUNK, *tail]
        y = torch.cat([x, x.new_zeros(1, *x.shape[1:])])[row]
        return y.reshape(n, chunks, CHUNK, hv, *tail).transpose(2, 3)

    q, k, v, g, beta = laid(q, dk), laid(k, dk), laid(v, dv), laid(s["g"]), laid(s["beta"])
    b = torch.cumsum(g, -1)
    decay = torch.exp(torch.clamp(b[..., :, None] - b[..., None, :], max=0.0))
    lower = torch.ones(CHUNK, CHUNK, device=dev).tril()
    a = beta[..., :, None] * decay * (k @ k.transpose(-1, -2)) * (lower - torch.eye(CHUNK, device=dev))
    inverse = unit_lower_inverse(a) * beta[..., None, :]
    attend = decay * (q @ k.transpose(-1, -2)) * lower
    last = torch.exp(b[..., -1:] - b)
    u0, w = inverse @ v, inverse @ (torch.exp(b)[..., None] * k)
    S = start_states(s)
    out = []
    for i in range(chunks):
        u = u0[:, i] - w[:, i] @ S.transpose(-1, -2)
        out.append(torch.exp(b[:, i])[..., None] * (q[:, i] @ S.transpose(-1, -2)) + attend[:, i] @ u)
        S = torch.exp(b[:, i, :, -1])[..., None, None] * S + (u * last[:, i][..., None]).transpose(-1, -2) @ k[:, i]
    o = torch.stack(out, 1).transpose(2, 3).reshape(n, chunks * CHUNK, hv, dv)
    s["out"].copy_(s["scale"] * o[inside])
    s["state"][s["slot"].long()] = S
    return {"out": s["out"], "state": s["state"]}


# ---- the definitions in 64 bits --------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers: compared for equality
    if case["op"] == "linear":
        return exact_linear(s)
    return exact_rule(s)


def exact_linear(s):
    c, k = s["case"], s["case"]["k"]
    w = s["w"][:, :k].double()
    if c["x"] == "int8":
        x, scale = s["x"][:, :k].double(), s["x_scale"].double()
    else:
        # the 8-bit values are defined by 32-bit steps (scale, its reciprocal, the product);
        # those are each one correctly rounded operation, made here on the host
        h = s["x"].float().cpu().numpy()
        top = np.abs(h).max(1).astype(np.float32)
        sc = np.where(top > 0, top / np.float32(127), np.float32(1)).astype(np.float32)
        scaled = (h * (np.float32(1) / sc)[:, None]).astype(np.float32).astype(np.float64)
        x = torch.from_numpy(np.clip(np.copysign(np.floor(np.abs(scaled) + 0.5), scaled), -127, 127)).to(w.device)
        scale = torch.from_numpy(sc.astype(np.float64)).to(w.device)
    y = torch.empty(c["m"], c["n"], dtype=torch.float64, device=w.device)
    for i in range(0, c["m"], 4096):
        y[i:i + 4096] = (x[i:i + 4096] @ w.T) * scale[i:i + 4096, None] * s["w_scale"].double()[None, :]
    return y


def exact_rule(s):
    """The recurrence, token by token, all requests and heads at once."""
    c = s["case"]
    hk, hv, dk, dv, lens = c["hk"], c["hv"], c["dk"], c["dv"], s["lens"]
    dev = s["q"].device
    slot = s["slot"].long()
    S = s["state"][slot].double()
    S[s["fresh"] != 0] = 0.0
    out = torch.zeros(s["q"].shape[0], hv, dv, dtype=torch.float64, device=dev)
    first = np.concatenate([[0], np.cumsum(lens)])[:-1]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])  # active requests are a prefix of this
    back = torch.tensor(order, device=dev)
    S = S[back]
    starts = torch.tensor([int(first[i]) for i in order], device=dev)
    sizes = [lens[i] for i in order]
    active = len(sizes)
    for t in range(max(lens)):
        while active and sizes[active - 1] <= t:
            active -= 1
        r = starts[:active] + t
        q, k, v = s["q"][r].double(), s["k"][r].double(), s["v"][r].double()
        if c["l2norm"]:
            q = q / (q.square().sum(-1, keepdim=True) + EPS).sqrt()
            k = k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()
        q = q[:, :, None].expand(active, hk, hv // hk, dk).reshape(active, hv, dk)
        k = k[:, :, None].expand(active, hk, hv // hk, dk).reshape(active, hv, dk)
        H = S[:active]
        H *= s["g"][r].double().exp()[:, :, None, None]
        u = s["beta"][r].double()[:, :, None] * (v - (H @ k[..., None])[..., 0])
        H += u[..., None] * k[:, :, None, :]
        out[r] = s["scale"] * (H @ q[..., None])[..., 0]
    state = s["state"].double()
    state[slot[back]] = S
    return {"out": out, "state": state}
