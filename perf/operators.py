"""Measured cases of the paged key-value cache operators: page planning, the
RoPE + cache append and the decode attention that reads the pages.

A case names an operator ("op") and its sizes.  ``run`` computes it in plain
torch operations, or -- with ``own`` set -- through the calls a user makes of
``krikil_rs_b200.kernels``.

Request lengths are the mid-points of an even division of low..high, in an
order drawn from the seed, so that a case's work does not depend on the seed.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one request a few tokens past its prompt: the batch-1 generation of the Pebble model, where latency counts
        attn("attn f32 batch 1", 1, 8, 8, 76, "f32", "f32", 16, 96, 96),
        # the decode attention workload [64, 8, 2048, 64] with positions spread over the cache
        attn("attn f32 64x8x2048x64", 64, 8, 8, 64, "f32", "f32", 16, 1, 2048),
        # the batched decode of 1024 sequences half way through their 256 new tokens
        attn("attn f32 1024x8x76", 1024, 8, 8, 76, "f32", "f32", 32, 128, 384),
        # a server's full decode batch of half-precision shared heads, some rows of the batch empty
        attn("attn bf16 128x32/8x128", 128, 32, 8, 128, "bf16", "bf16", 64, 0, 8192),
        # one very long document, few heads: the cache's length is all there is to split
        attn("attn f16 1x16/2x256 long", 1, 16, 2, 256, "f16", "f16", 16, 131071, 131071),
        # float32 activations over a half-size cache, with a sliding window
        attn("attn f32 on bf16 window", 48, 12, 4, 80, "f32", "bf16", 128, 1, 6000, window=1000),
        # one new token of one request
        append("append f32 batch 1", 1, 0, 8, 8, 76, 76, "f32", "f32", 16, 2048),
        # the batched decode's append: one token of each of 1024 sequences
        append("append f32 1024x8x76", 1024, 0, 8, 8, 76, 76, "f32", "f32", 32, 2048),
        # a prefill chunk of a long-context model, its last rows padding
        append("append bf16 16384x32/8x128", 16321, 63, 32, 8, 128, 128, "bf16", "bf16", 64, 1000000),
        # float32 activations into a half-size cache, part of each head rotated
        append("append f32 to f16 2000x12/4x80", 2000, 7, 12, 4, 80, 40, "f32", "f16", 16, 32768),
        # a decode step's plan: one token for each of 1024 requests, some of them finished and released
        plan("plan decode 1024", 1024, 1, 2048, 1, 1, 16, done=32),
        # prompts admitted at once: ragged new tokens on top of shared prefixes
        plan("plan prompts 61", 61, 0, 4096, 1, 8191, 64, done=0),
    ]


def attn(name, batch, hq, hkv, dh, act, cache, page, low, high, window=0):
    return {"name": name, "op": "attn", "batch": batch, "hq": hq, "hkv": hkv, "dh": dh, "act": act, "cache": cache,
            "page": page, "low": low, "high": high, "window": window}


def append(name, tokens, pad, hq, hkv, dh, rot, act, cache, page, far):
    return {"name": name, "op": "append", "tokens": tokens, "pad": pad, "hq": hq, "hkv": hkv, "dh": dh, "rot": rot,
            "act": act, "cache": cache, "page": page, "far": far}


def plan(name, batch, low, high, new_low, new_high, page, done):
    return {"name": name, "op": "plan", "batch": batch, "low": low, "high": high, "new_low": new_low,
            "new_high": new_high, "page": page, "done": done}


def draw(rng):
    def spread(a, b):  # whole numbers evenly spread over their logarithm
        return max(a, min(b, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))

    op = rng.choice(["attn", "attn", "append", "plan"])
    page = rng.choice([8, 16, 32, 64, 128])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    hkv = rng.choice([1, 2, 4, 5, 8])
    hq = hkv * rng.choice([1, 1, 2, 3, 4, 7, 8])
    dh = rng.choice([64, 64, 76, 80, 96, 128, 128, 192, 256])
    if op == "attn":
        row = 2 * hkv * dh * SIZE[cache]
        high = spread(1, 131072)
        batch = spread(1, max(1, min(1024, int(1.5e9 / row / high))))
        # the plain form widens every row to the longest one, in 32 bits and once per query head
        batch = max(1, min(batch, int(6e9 / (high * (2 * hkv * dh + 3 * hq) * 4))))
        low = rng.choice([0, 1, high // 2, high])
        window = rng.choice([0, 0, 0, spread(1, max(1, high))])
        c = attn("", batch, hq, hkv, dh, act, cache, page, low, high, window)
    elif op == "append":
        rot = rng.choice([dh, dh, dh // 2 // 2 * 2])
        c = append("", spread(1, 16384), rng.choice([0, 0, spread(1, 64)]), hq, hkv, dh, rot, act, cache, page,
                   rng.choice([2048, 32768, 1000000]))
        c["tokens"] = min(c["tokens"], max(1, int(2e8 / ((hq + hkv) * dh * 4))))
    else:
        batch = spread(1, 2048)
        new_high = spread(1, max(1, 400000 // batch))
        c = plan("", batch, 0, spread(1, 8192), rng.choice([0, 1, new_high]), new_high, page,
                 rng.choice([0, 0, batch // 4]))
    del c["name"]
    return c


# ------------------------------------------------------------------ the inputs
def lengths(low, high, n):
    return [low + int((high - low) * (i + 0.5) / n + 0.5) if high > low else high for i in range(n)]


def pages_of(n, page):
    return (n + page - 1) // page


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"attn": prepare_attn, "append": prepare_append, "plan": prepare_plan}[case["op"]](case, g)


def shuffled(values, g):
    order = torch.randperm(len(values), generator=g, device=DEV)
    return torch.tensor(values, device=DEV, dtype=torch.int32)[order]


def normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def page_table(lens, width, page, num_pages, g):
    """Distinct pages in a random order for every request's rows; 0 where a row ends."""
    need = (lens + (page - 1)) // page
    used = torch.arange(width, device=DEV)[None, :] < need[:, None]
    rank = (torch.cumsum(used.reshape(-1).int(), 0) - 1).reshape(used.shape)
    order = torch.randperm(num_pages, generator=g, device=DEV)
    return torch.where(used, order[rank.clamp_min(0)], torch.zeros_like(rank)).int().contiguous()


def prepare_attn(c, g):
    values = lengths(c["low"], c["high"], c["batch"])
    lens = shuffled(values, g)
    width = max(1, pages_of(max(values), c["page"]))
    num_pages = max(1, sum(pages_of(n, c["page"]) for n in values))
    shape = (num_pages, c["page"], c["hkv"], c["dh"])
    return {"case": c, "lens": lens, "max_len": max(values),
            "table": page_table(lens, width, c["page"], num_pages, g),
            "q": normal(g, TYPES[c["act"]], c["batch"], c["hq"], c["dh"]),
            "kc": normal(g, TYPES[c["cache"]], *shape), "vc": normal(g, TYPES[c["cache"]], *shape)}


def prepare_append(c, g):
    n, rows = c["tokens"], c["tokens"] + c["pad"]
    num_pages = pages_of(n, c["page"]) + 3
    act, cache = TYPES[c["act"]], TYPES[c["cache"]]
    # q, k and v as a projection leaves them: slices of one packed row
    packed = normal(g, act, rows, (c["hq"] + 2 * c["hkv"]) * c["dh"])
    q, k, v = (x.unflatten(1, (-1, c["dh"])) for x in
               packed.split([c["hq"] * c["dh"], c["hkv"] * c["dh"], c["hkv"] * c["dh"]], dim=1))
    slots = torch.full((rows,), -1, device=DEV, dtype=torch.int32)
    slots[:n] = torch.randperm(num_pages * c["page"], generator=g, device=DEV)[:n].int()
    positions = torch.randint(0, c["far"], (rows,), generator=g, device=DEV, dtype=torch.int32)
    shape = (num_pages, c["page"], c["hkv"], c["dh"])
    return {"case": c, "q": q, "k": k, "v": v, "slots": slots, "positions": positions,
            "q_out": torch.zeros(rows, c["hq"], c["dh"], device=DEV, dtype=act),
            "kc": torch.zeros(shape, device=DEV, dtype=cache), "vc": torch.zeros(shape, device=DEV, dtype=cache)}


def plan_sizes(c):
    """What a request holds and adds, paired before they are shuffled; the first `done` of them are finished."""
    held = lengths(c["low"], c["high"], c["batch"])
    new = lengths(c["new_low"], c["new_high"], c["batch"])
    new = [0 if i < c["done"] else new[(i * 7) % c["batch"]] for i in range(c["batch"])]
    return held, new


def prepare_plan(c, g):
    held, new = plan_sizes(c)
    order = torch.randperm(c["batch"], generator=g, device=DEV)
    lens = torch.tensor(held, device=DEV, dtype=torch.int32)[order]
    fresh = torch.tensor(new, device=DEV, dtype=torch.int32)[order]
    done = (torch.arange(c["batch"], device=DEV) < c["done"])[order]
    page = c["page"]
    in_use = sum(pages_of(n, page) for n in held)
    wanted = sum(pages_of(a + b, page) - pages_of(a, page) for a, b in zip(held, new))
    back = sum(pages_of(n, page) for n in held[:c["done"]])
    num_pages = in_use + wanted + 17
    width = max(1, max(pages_of(a + b, page) for a, b in zip(held, new)))
    order = torch.randperm(num_pages, generator=g, device=DEV).int()
    need = (lens + (page - 1)) // page
    used = torch.arange(width, device=DEV)[None, :] < need[:, None]
    rank = (torch.cumsum(used.reshape(-1).int(), 0) - 1).reshape(used.shape)
    table = torch.where(used, order[rank.clamp_min(0)], -1).int().contiguous()
    free = torch.full((num_pages,), -1, device=DEV, dtype=torch.int32)
    free[: num_pages - in_use] = order[in_use:]
    tokens = sum(new)
    return {"case": c, "lens": lens, "new": fresh, "done": done, "table": table, "free": free,
            "count": torch.tensor([num_pages - in_use], device=DEV, dtype=torch.int32),
            "rows": max(1, (tokens + 7) // 8 * 8),  # the step's padded token count
            "tokens": tokens, "wanted": wanted, "back": back}


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        from krikil_rs_b200 import kernels as K
        return {"attn": own_attn, "append": own_append, "plan": own_plan}[op](state, K)
    return {"attn": plain_attn, "append": plain_append, "plan": plain_plan}[op](state)


def own_attn(s, K):
    return K.attn_decode_paged(s["q"], s["kc"], s["vc"], s["table"], s["lens"], window=s["case"]["window"],
                               max_len=s["max_len"], return_lse=True)


def own_append(s, K):
    K.rope_kv_append_paged(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["positions"],
                           rot_dim=s["case"]["rot"], q_out=s["q_out"])
    return s["q_out"], s["kc"], s["vc"]


def own_plan(s, K):
    lens, count, back = s["lens"], s["count"], None
    if s["case"]["done"]:
        lens, count, back = K.kv_page_release(s["done"], lens, s["table"], s["free"], count, s["case"]["page"])
    lens, count, cu, positions, slots, status = K.kv_page_plan(s["new"], lens, s["table"], s["free"], count,
                                                               s["case"]["page"], s["rows"])
    out = {"lens": lens, "count": count, "cu": cu, "positions": positions, "slots": slots, "status": status,
           "table": s["table"], "free": s["free"]}
    return out if back is None else dict(out, released=back)


def plain_attn(s):
    c = s["case"]
    b, hq, hkv, dh = c["batch"], c["hq"], c["hkv"], c["dh"]
    at = torch.arange(max(1, s["max_len"]), device=DEV)
    lens = s["lens"].long()[:, None]
    seen = at[None, :] < lens
    if c["window"]:
        seen = seen & (at[None, :] >= lens - c["window"])
    pages, offs = s["table"].long()[:, at // c["page"]], (at % c["page"])[None, :].expand(b, -1)
    k, v = s["kc"][pages, offs].float(), s["vc"][pages, offs].float()  # [b, keys, hkv, dh]
    v = torch.where(seen[:, :, None, None], v, 0.0)
    q = s["q"].float().reshape(b, hkv, hq // hkv, dh)
    x = torch.einsum("bhgd,blhd->bhgl", q, k) * (1.0 / math.sqrt(dh))
    x = torch.where(seen[:, None, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("bhgl,blhd->bhgd", p, v) / torch.where(total == 0, 1.0, total)
    lse = top + torch.log(total)
    return out.reshape(b, hq, dh).to(s["q"].dtype), lse.reshape(b, hq)


def plain_append(s):
    c, n = s["case"], s["case"]["tokens"]
    half = c["rot"] // 2
    turn = 10000.0 ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / c["rot"])
    angle = s["positions"][:n].double()[:, None] * turn[None, :]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]

    def rotated(x):
        x = x.float()
        a, b = x[..., :half], x[..., half:c["rot"]]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., c["rot"]:]], dim=-1)

    page, off = s["slots"][:n].long() // c["page"], s["slots"][:n].long() % c["page"]
    s["kc"][page, off] = rotated(s["k"][:n]).to(s["kc"].dtype)
    s["vc"][page, off] = s["v"][:n].to(s["vc"].dtype)
    s["q_out"][:n] = rotated(s["q"][:n]).to(s["q_out"].dtype)
    return s["q_out"], s["kc"], s["vc"]


def plain_plan(s):
    c, page = s["case"], s["case"]["page"]
    lens, count, table, free = s["lens"].long(), s["count"].long(), s["table"], s["free"]
    out = {}
    if c["done"]:
        held = torch.where(s["done"], (lens + page - 1) // page, 0)
        start = torch.cumsum(held, 0) - held
        row = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), held, output_size=s["back"])
        nth = torch.arange(s["back"], device=DEV)
        free[count + nth] = table[row, nth - start[row]]
        lens = torch.where(s["done"], 0, lens)
        count = count + held.sum()
        out["released"] = torch.zeros(1, device=DEV, dtype=torch.int32)
    new = s["new"].long()
    have = (lens + page - 1) // page
    need = (lens + new + page - 1) // page - have
    start = torch.cumsum(need, 0) - need
    row = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), need, output_size=s["wanted"])
    nth = torch.arange(s["wanted"], device=DEV)
    table[row, have[row] + nth - start[row]] = free[count - 1 - nth]
    cu = torch.cat([torch.zeros(1, device=DEV, dtype=torch.int64), torch.cumsum(new, 0)])
    row = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), new, output_size=s["tokens"])
    at = lens[row] + torch.arange(s["tokens"], device=DEV) - cu[row]
    slots = torch.full((s["rows"],), -1, device=DEV, dtype=torch.int32)
    slots[: s["tokens"]] = (table[row, at // page].long() * page + at % page).int()
    positions = torch.zeros(s["rows"], device=DEV, dtype=torch.int32)
    positions[: s["tokens"]] = at.int()
    return dict(out, lens=(lens + new).int(), count=(count - need.sum()).int(), cu=cu.int(), positions=positions,
                slots=slots, status=torch.zeros(1, device=DEV, dtype=torch.int32), table=table, free=free)


# ------------------------------------------------------------------ the work
def work(c):
    if c["op"] == "attn":
        n = [min(x, c["window"]) if c["window"] else x for x in lengths(c["low"], c["high"], c["batch"])]
        keys = sum(n)
        rows = c["batch"] * c["hq"]
        return {"bytes": keys * c["hkv"] * c["dh"] * 2 * SIZE[c["cache"]] + rows * c["dh"] * 2 * SIZE[c["act"]] + rows * 4
                + 4 * sum(pages_of(x, c["page"]) for x in n) + 4 * c["batch"],
                "flops": keys * c["hq"] * (4 * c["dh"] + 4)}
    if c["op"] == "append":
        heads = c["tokens"] * c["dh"]
        return {"bytes": heads * (2 * c["hq"] + 2 * c["hkv"]) * SIZE[c["act"]] + heads * 2 * c["hkv"] * SIZE[c["cache"]]
                + 4 * (c["tokens"] + c["pad"]) + 4 * c["tokens"],
                "flops": 3 * c["tokens"] * (c["hq"] + c["hkv"]) * c["rot"]}
    held, new = plan_sizes(c)
    page = c["page"]
    wanted = sum(pages_of(a + b, page) - pages_of(a, page) for a, b in zip(held, new))
    back = sum(pages_of(n, page) for n in held[:c["done"]])
    rows = max(1, (sum(new) + 7) // 8 * 8)
    return {"bytes": 8 * rows + 8 * (wanted + back) + 16 * c["batch"] + 4 * c["batch"] * (c["done"] > 0) + 24,
            "flops": 4 * rows + 8 * c["batch"]}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return exact_attn(s)
    if case["op"] == "append":
        return exact_append(s)
    return None


def exact_attn(s):
    """softmax(q K^T / sqrt(dh)) V request by request, straight from the definition."""
    c = s["case"]
    out = torch.zeros(c["batch"], c["hq"], c["dh"], device=DEV, dtype=torch.float64)
    lse = torch.full((c["batch"], c["hq"]), -math.inf, device=DEV, dtype=torch.float64)
    share = c["hq"] // c["hkv"]
    for i, n in enumerate(s["lens"].tolist()):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        rows = s["table"][i, : pages_of(n, c["page"])].long()
        k = s["kc"][rows].flatten(0, 1)[first:n].double()
        v = s["vc"][rows].flatten(0, 1)[first:n].double()
        for h in range(c["hkv"]):
            q = s["q"][i, h * share:(h + 1) * share].double()
            x = q @ k[:, h].T / math.sqrt(c["dh"])
            lse[i, h * share:(h + 1) * share] = torch.logsumexp(x, 1)
            out[i, h * share:(h + 1) * share] = torch.softmax(x, 1) @ v[:, h]
    return out, lse


def exact_append(s):
    """Each pair (x_i, x_{i + rot/2}) as a complex number, turned by position / 10000^(2 i / rot)."""
    c, n = s["case"], s["case"]["tokens"]
    half = c["rot"] // 2
    rate = torch.exp(torch.arange(half, device=DEV, dtype=torch.float64) * (-2.0 / c["rot"] * math.log(10000.0)))
    turn = torch.polar(torch.ones(n, half, device=DEV, dtype=torch.float64),
                       torch.outer(s["positions"][:n].double(), rate))

    def rotated(x):
        x = x[:n].double()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn[:, None, :]
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], dim=-1)

    kc, vc, q = s["kc"].double(), s["vc"].double(), s["q_out"].double()
    where = s["slots"][:n].long()
    kc.view(-1, c["hkv"], c["dh"])[where] = rotated(s["k"])
    vc.view(-1, c["hkv"], c["dh"])[where] = s["v"][:n].double()
    q[:n] = rotated(s["q"])
    return q, kc, vc
