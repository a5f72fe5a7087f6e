"""Measured cases of the operators of recurrent layers that serve many requests --
the short causal convolution and the selective state space scan, for packed
prompts and for single tokens, over a pool of state slots -- and of the log
probabilities with which a server answers.

A case names an operator ("op") and its sizes.  ``run`` computes it in plain
torch operations, or -- with ``own`` set -- through the calls a user makes of
``krikil_rs_b200.kernels``.

Request lengths are the mid-points of an even division of low..high, in an
order drawn from the seed, so that a case's work does not depend on the seed.
Every pass reads its requests' states from slots that it does not write (a
shared prefix that several requests continue, drafted tokens that may be taken
back), so that a pass finds what the one before it found.
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
        # the convolution channels of one prompt of the Pebble model, as its batch-1 generation has it
        conv("conv f32 prompt 32x1472", 1, 32, 32, 0, 1472, 4, "f32", 0),
        # a prefill step of a server: ragged prompts, half of them continuing, padding rows behind them
        conv("conv bf16 64 prompts x8192", 64, 0, 511, 17, 8192, 4, "bf16", 32),
        # one token of one request
        conv_step("conv step f32 1x1472", 1, 0, 1472, 4, "f32"),
        # a server's decode batch, some of its rows empty
        conv_step("conv step bf16 509x8192", 509, 3, 8192, 4, "bf16"),
        # one short prompt of a model of Pebble's width, where latency counts
        scan("scan f32 prompt 32x1216", 1, 32, 32, 0, 1216, 16, 1, "f32", 0),
        # one long prompt of a narrow model: few channels to share out, and a long way to go
        scan("scan f16 8192x1536", 1, 8192, 8192, 0, 1536, 16, 1, "f16", 1),
        # a prefill step of a server: ragged prompts, half of them continuing, padding rows behind them
        scan("scan bf16 64 prompts x5120", 64, 0, 511, 17, 5120, 16, 1, "bf16", 32),
        # one token of one request
        step("step f32 1x1216", 1, 0, 1216, 16, 1, "f32"),
        # a server's decode batch, some of its rows empty
        step("step bf16 253x5120", 253, 3, 5120, 16, 1, "bf16"),
        # one pick of a long vocabulary, with the alternatives that a client may ask for
        logprobs("logprobs f32 1x131072 top 20", 1, 131072, 1, 20, "f32"),
        # the batched decode of 1024 sequences over the Pebble vocabulary
        logprobs("logprobs f32 1024x2048 top 5", 1024, 2048, 1, 5, "f32"),
        # the rows of scored prompts: each one's next token and the best other
        logprobs("logprobs bf16 4096x50001", 4096, 50001, 1, 1, "bf16"),
    ]


def conv(name, requests, low, high, pad, channels, width, act, continued):
    return {"name": name, "op": "conv", "requests": requests, "low": low, "high": high, "pad": pad,
            "channels": channels, "width": width, "act": act, "continued": continued}


def conv_step(name, rows, pad, channels, width, act):
    return {"name": name, "op": "conv step", "rows": rows, "pad": pad, "channels": channels, "width": width,
            "act": act}


def scan(name, requests, low, high, pad, channels, n, groups, act, continued):
    return {"name": name, "op": "scan", "requests": requests, "low": low, "high": high, "pad": pad,
            "channels": channels, "n": n, "groups": groups, "act": act, "continued": continued}


def step(name, rows, pad, channels, n, groups, act):
    return {"name": name, "op": "step", "rows": rows, "pad": pad, "channels": channels, "n": n, "groups": groups,
            "act": act}


def logprobs(name, rows, vocab, asked, top, act):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "asked": asked, "top": top, "act": act}


def draw(rng):
    def spread(a, b):  # whole numbers evenly spread over their logarithm
        return max(a, min(b, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))

    op = rng.choice(["conv", "conv step", "scan", "scan", "step", "logprobs", "logprobs"])
    act = rng.choice(["f32", "f16", "bf16"])
    width = rng.choice([2, 3, 4, 4, 4])
    groups = rng.choice([1, 1, 1, 2, 4])
    n = rng.choice([4, 8, 16, 16, 16, 24, 32, 64])
    if op == "logprobs":
        vocab = spread(256, 262144)
        rows = min(spread(1, 8192), max(1, 200000000 // vocab))
        return unnamed(logprobs("", rows, vocab, rng.choice([1, 1, 2, 5]), rng.choice([0, 1, 5, 20]), act))
    if op == "conv step":
        return unnamed(conv_step("", spread(1, 512), rng.choice([0, 0, 5]), spread(32, 8192), width, act))
    if op == "step":
        channels = spread(64, 5120) // groups * groups
        rows = min(spread(1, 512), max(1, 20000000 // (channels * n)))
        return unnamed(step("", rows, rng.choice([0, 0, 5]), channels, n, groups, act))
    requests = spread(1, 64)
    tokens = spread(requests, 16000)
    if op == "conv":
        channels = spread(32, 8192)
        tokens = max(requests, min(tokens, 64000000 // channels))
    else:
        channels = spread(64, 5120) // groups * groups
        tokens = max(requests, min(tokens, 600000000 // (channels * n)))
    high = max(1, tokens // requests)
    low = rng.choice([0, high // 2, high])
    pad, continued = rng.choice([0, 0, 17]), rng.choice([0, requests // 2, requests])
    if op == "conv":
        return unnamed(conv("", requests, low, high, pad, channels, width, act, continued))
    return unnamed(scan("", requests, low, high, pad, channels, n, groups, act, continued))


def unnamed(case):
    return {key: value for key, value in case.items() if key != "name"}


# ------------------------------------------------------------------ the inputs
def lengths(c):
    low, high, n = c["low"], c["high"], c["requests"]
    return [low + int((high - low) * (i + 0.5) / n + 0.5) if high > low else high for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"conv": prepare_conv, "conv step": prepare_conv, "scan": prepare_scan, "step": prepare_scan,
            "logprobs": prepare_logprobs}[case["op"]](case, g)


def normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def requests_of(c, g):
    """Where each packed request's rows begin (cu), where its state goes (slots) and where it comes from (init: -1,
    nothing, for those that begin); for single tokens a row a request, those behind the last one without a slot."""
    single = "rows" in c
    count, pad = (c["rows"], c["pad"]) if single else (c["requests"], 0)
    order = torch.randperm(2 * count + 1, generator=g, device=DEV).int()
    slots = torch.full((count + pad,), -1, device=DEV, dtype=torch.int32)
    init = torch.full((count + pad,), -1, device=DEV, dtype=torch.int32)
    slots[:count], init[:count] = order[:count], order[count:2 * count]
    s = {"case": c, "slots": slots, "init": init, "pool": 2 * count + 1, "rows": count + pad}
    if not single:
        values = lengths(c)
        lens = torch.tensor(values, device=DEV)[torch.randperm(count, generator=g, device=DEV)]
        init[torch.randperm(count, generator=g, device=DEV)[c["continued"]:]] = -1
        s["cu"] = torch.cat([lens.new_zeros(1), torch.cumsum(lens, 0)]).int()
        s["tokens"] = sum(values)
        s["rows"] = max(1, s["tokens"] + c["pad"])
    return s


def prepare_conv(c, g):
    s, ch, act = requests_of(c, g), c["channels"], TYPES[c["act"]]
    # x as a projection leaves it, with the gate beside it
    s["x"] = normal(g, act, s["rows"], 2 * ch)[:, :ch]
    s["weight"] = 0.5 * normal(g, torch.float32, ch, c["width"])
    s["bias"] = 0.1 * normal(g, torch.float32, ch)
    s["state"] = normal(g, act, s["pool"], c["width"] - 1, ch)
    s["out"] = torch.zeros(s["rows"], ch, device=DEV, dtype=act)
    return s


def prepare_scan(c, g):
    s, ch, n, act = requests_of(c, g), c["channels"], c["n"], TYPES[c["act"]]
    gn, rank = c["groups"] * n, (ch + 15) // 16
    s["x"] = normal(g, act, s["rows"], ch)
    s["z"] = normal(g, act, s["rows"], 2 * ch)[:, ch:]  # the other half of the projection that x came from
    # B and C as slices of one projection, beside the step widths' low rank
    low = normal(g, act, s["rows"], rank + 2 * gn)
    s["b"] = low[:, rank:rank + gn].unflatten(1, (c["groups"], n))
    s["c"] = low[:, rank + gn:].unflatten(1, (c["groups"], n))
    s["dt"] = 0.5 * normal(g, act, s["rows"], ch)
    # step widths of 0.001 to 0.1 and decays of about 1 .. n, the usual beginnings of such layers
    width = torch.exp(math.log(1e-3) + (math.log(1e-1) - math.log(1e-3))
                      * torch.rand(ch, generator=g, device=DEV, dtype=torch.float64))
    s["dt_bias"] = torch.log(torch.expm1(width)).float()
    s["a"] = -(torch.arange(1, n + 1, device=DEV)[None, :] * torch.exp(0.2 * normal(g, torch.float32, ch, n)))
    s["d"] = 1.0 + 0.1 * normal(g, torch.float32, ch)
    s["state"] = normal(g, torch.float32, s["pool"], ch, n)
    s["out"] = torch.zeros(s["rows"], ch, device=DEV, dtype=act)
    return s


def prepare_logprobs(c, g):
    logits = normal(g, TYPES[c["act"]], c["rows"], c["vocab"])
    logits *= 3.0
    tokens = torch.randint(0, c["vocab"], (c["rows"], c["asked"]), generator=g, device=DEV, dtype=torch.int32)
    return {"case": c, "logits": logits, "tokens": tokens}


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        from krikil_rs_b200 import kernels as K
        return {"conv": own_conv, "conv step": own_conv_step, "scan": own_scan, "step": own_step,
                "logprobs": own_logprobs}[op](state, K)
    return {"conv": plain_conv, "conv step": plain_conv_step, "scan": plain_scan, "step": plain_step,
            "logprobs": plain_logprobs}[op](state)


def own_conv(s, K):
    K.causal_conv(s["x"], s["weight"], s["cu"], bias=s["bias"], state=s["state"], slots=s["slots"], init=s["init"],
                  out=s["out"])
    return s["out"], s["state"]


def own_conv_step(s, K):
    K.causal_conv_step(s["x"], s["weight"], s["state"], s["slots"], bias=s["bias"], init=s["init"], out=s["out"])
    return s["out"], s["state"]


def own_scan(s, K):
    K.selective_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], s["cu"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                     state=s["state"], slots=s["slots"], init=s["init"], out=s["out"])
    return s["out"], s["state"]


def own_step(s, K):
    K.selective_step(s["x"], s["dt"], s["a"], s["b"], s["c"], s["state"], s["slots"], d=s["d"], z=s["z"],
                     dt_bias=s["dt_bias"], init=s["init"], out=s["out"])
    return s["out"], s["state"]


def own_logprobs(s, K):
    return K.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])


def silu(x):
    return x / (1.0 + torch.exp(-x))


def softplus(x):
    return torch.where(x > 20.0, x, torch.log1p(torch.exp(x.clamp(max=20.0))))


def request_rows(s):
    """The request of each of the packed rows, and its row within it."""
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    owner = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), lens, output_size=s["tokens"])
    return owner, torch.arange(s["tokens"], device=DEV) - s["cu"].long()[owner]


def begun(s, count):
    """The states that the requests continue, in 32 bits: zeros for those that begin."""
    init = s["init"][:count].long()
    old = s["state"][init.clamp_min(0)].float()
    return torch.where((init >= 0)[:, None, None], old, 0.0)


def plain_conv(s):
    c, count, width, rows = s["case"], s["case"]["requests"], s["case"]["width"], s["tokens"]
    owner, at = request_rows(s)
    first = torch.arange(count, device=DEV) * (width - 1)
    # the requests' old rows in front of the new ones: row r of request i is at old + r, or among its old ones
    full = torch.cat([begun(s, count).flatten(0, 1), s["x"][:rows].float()])
    back = torch.arange(width, device=DEV) - (width - 1)

    def source(owner, at, start):
        here = at[:, None] + back[None, :]
        return torch.where(here < 0, first[owner][:, None] + width - 1 + here, count * (width - 1) + start[:, None] + here)

    start = s["cu"].long()[:-1]
    taps = full[source(owner, at, start[owner])]  # [rows, width, channels]
    y = (taps * s["weight"].T[None]).sum(1) + s["bias"]
    s["out"][:rows] = silu(y).to(s["out"].dtype)
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    last = full[source(torch.arange(count, device=DEV), lens - 1, start)[:, 1:]]
    s["state"][s["slots"].long()] = last.to(s["state"].dtype)
    return s["out"], s["state"]


def plain_conv_step(s):
    count = s["case"]["rows"]
    taps = torch.cat([begun(s, count), s["x"][:count].float()[:, None]], dim=1)
    y = (taps * s["weight"].T[None]).sum(1) + s["bias"]
    s["out"][:count] = silu(y).to(s["out"].dtype)
    s["state"][s["slots"][:count].long()] = taps[:, 1:].to(s["state"].dtype)
    return s["out"], s["state"]


def recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = 0 over the first dimension: the odd rows from pairs, the even ones from
    the odd."""
    if a.shape[0] == 1:
        return b
    even, odd = slice(0, a.shape[0] - 1, 2), slice(1, None, 2)
    h = torch.empty_like(b)
    h[odd] = recurrence(a[odd] * a[even], torch.addcmul(b[odd], a[odd], b[even]))
    h[0] = b[0]
    h[2::2] = torch.addcmul(b[2::2], a[2::2], h[1:-1:2])
    return h


def widened(s, name, rows):
    """B or C of every channel: [rows, channels, n]."""
    c = s["case"]
    return s[name][:rows].float().repeat_interleave(c["channels"] // c["groups"], dim=1)


def gated(s, y, rows):
    y = y + s["d"] * s["x"][:rows].float()
    s["out"][:rows] = (y * silu(s["z"][:rows].float())).to(s["out"].dtype)


def plain_scan(s):
    count, rows = s["case"]["requests"], s["tokens"]
    h0 = begun(s, count)
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    if rows:
        owner, at = request_rows(s)
        delta = softplus(s["dt"][:rows].float() + s["dt_bias"])
        a = torch.exp(delta[:, :, None] * s["a"])
        b = (delta * s["x"][:rows].float())[:, :, None] * widened(s, "b", rows)
        # a request's first row takes its old state and forgets the row before it
        begins = (s["cu"].long()[:-1]).clamp(max=rows - 1)[lens > 0]
        b[begins] += a[begins] * h0[lens > 0]
        a[begins] = 0.0
        h = recurrence(a, b)
        del a, b
        gated(s, (h * widened(s, "c", rows)).sum(2), rows)
        h0 = torch.where((lens > 0)[:, None, None], h[(s["cu"].long()[1:] - 1).clamp_min(0)], h0)
    s["state"][s["slots"].long()] = h0
    return s["out"], s["state"]


def plain_step(s):
    rows = s["case"]["rows"]
    delta = softplus(s["dt"][:rows].float() + s["dt_bias"])
    h = torch.exp(delta[:, :, None] * s["a"]) * begun(s, rows)
    h = h + (delta * s["x"][:rows].float())[:, :, None] * widened(s, "b", rows)
    gated(s, (h * widened(s, "c", rows)).sum(2), rows)
    s["state"][s["slots"][:rows].long()] = h
    return s["out"], s["state"]


def plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    shifted = x - x.amax(1, keepdim=True)
    p = torch.exp(shifted)
    total = p.sum(1, keepdim=True)
    log_total = torch.log(total)
    given = torch.gather(shifted, 1, s["tokens"].long()) - log_total
    entropy = log_total[:, 0] - (p * shifted).sum(1) / total[:, 0]
    # the order of the logits as whole numbers, the lower index first among equal ones (-0 is 0)
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    key = bits * 2 ** 31 + (2 ** 31 - 1 - torch.arange(c["vocab"], device=DEV))
    ids = torch.topk(key, c["top"], dim=1).indices
    return given, entropy, ids.int(), torch.gather(shifted, 1, ids) - log_total


# ------------------------------------------------------------------ the work
def work(c):
    size = SIZE[c["act"]]
    if c["op"] == "logprobs":
        values = c["rows"] * c["vocab"]
        return {"bytes": values * size + c["rows"] * (8 * c["asked"] + 4 + 8 * c["top"]), "flops": 6 * values}
    single = "rows" in c
    tokens = c["rows"] if single else sum(lengths(c))
    requests, continued = (c["rows"], c["rows"]) if single else (c["requests"], c["continued"])
    ch = c["channels"]
    if c["op"] in ("conv", "conv step"):
        return {"bytes": 2 * tokens * ch * size + (requests + continued) * (c["width"] - 1) * ch * size
                + 4 * ch * (c["width"] + 1), "flops": tokens * ch * (2 * c["width"] + 5)}
    return {"bytes": 4 * tokens * ch * size + 2 * tokens * c["groups"] * c["n"] * size
            + 4 * (requests + continued) * ch * c["n"] + 4 * ch * (c["n"] + 2),
            "flops": tokens * ch * (7 * c["n"] + 14)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": exact_conv, "conv step": exact_conv, "scan": exact_scan, "step": exact_scan,
            "logprobs": exact_logprobs}[case["op"]](s)


def spans(s):
    """(first row, row behind the last, slot, slot of the old state) of each request."""
    cu = range(s["case"]["rows"] + 1) if "rows" in s["case"] else s["cu"].tolist()
    return list(zip(cu[:-1], cu[1:], s["slots"].tolist(), s["init"].tolist()))


def exact_conv(s):
    """Each request by itself: its old rows, then its new ones, under the window of taps."""
    width = s["case"]["width"]
    out, state = s["out"].double(), s["state"].double()
    old, w = state.clone(), s["weight"].double()
    for i, j, slot, init in spans(s):
        rows = torch.cat([old[init] if init >= 0 else torch.zeros_like(old[0]), s["x"][i:j].double()])
        y = s["bias"].double().expand(j - i, -1)
        for k in range(width):
            y = y + w[:, k] * rows[k:k + j - i]
        out[i:j] = y * torch.sigmoid(y)
        state[slot] = rows[j - i:]
    return out, state


def exact_scan(s):
    """Each request by itself, row after row."""
    c = s["case"]
    out, state = s["out"].double(), s["state"].double()
    old, share = state.clone(), c["channels"] // c["groups"]
    for i, j, slot, init in spans(s):
        h = old[init] if init >= 0 else torch.zeros_like(old[0])
        x = s["x"][i:j].double()
        delta = torch.nn.functional.softplus(s["dt"][i:j].double() + s["dt_bias"].double(), threshold=50.0)
        z, a, d = s["z"][i:j].double(), s["a"].double(), s["d"].double()
        bm = s["b"][i:j].double().repeat_interleave(share, dim=1)
        cm = s["c"][i:j].double().repeat_interleave(share, dim=1)
        for t in range(j - i):
            h = torch.exp(a * delta[t, :, None]) * h + bm[t] * (delta[t] * x[t])[:, None]
            y = (h * cm[t]).sum(1) + d * x[t]
            out[i + t] = y * (z[t] * torch.sigmoid(z[t]))
        state[slot] = h
    return out, state


def exact_logprobs(s):
    """The ids, whole numbers, are left to the plain form."""
    given, entropy, best = [], [], []
    for rows, tokens in zip(s["logits"].split(64), s["tokens"].split(64)):
        lp = torch.log_softmax(rows.double(), 1)
        given.append(torch.gather(lp, 1, tokens.long()))
        entropy.append(-(lp.exp() * lp).sum(1))
        best.append(torch.sort(lp, dim=1, descending=True).values[:, :s["case"]["top"]])
    return torch.cat(given), torch.cat(entropy), None, torch.cat(best)
