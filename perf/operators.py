"""Cases of the 8-bit paged KV cache operators: append, attention, eviction.

One layer of the cache is ``codes`` [pages, Hkv, 2, 16, D] (int8 or float8_e4m3fn,
K then V), ``scales`` fp32 [pages, Hkv, 2] (one for each block of 16 tokens, head
and K / V) and ``mass`` fp32 [pages, Hkv, 16] (accumulated attention weight).

``run`` computes a case in elementary torch operations in 32 bits, or, with ``own``
set, through ``complexity_framework_b200.ops.paged8``.
"""
import math

import torch

own = False

PAGE = 16
LEVELS = {"int8": 127.0, "fp8": 448.0}
STORE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


# ------------------------------------------------------------------- the cases
def _append(name, code, seqs, q, kv_min, kv_max, hkv, d):
    return {"name": name, "op": "append", "code": code, "seqs": seqs, "q": q, "kv_min": kv_min,
            "kv_max": kv_max, "hkv": hkv, "d": d}


def _attend(name, code, seqs, q, kv_min, kv_max, hq, hkv, d, mass=False, empty=0):
    return {"name": name, "op": "attend", "code": code, "seqs": seqs, "q": q, "kv_min": kv_min,
            "kv_max": kv_max, "hq": hq, "hkv": hkv, "d": d, "mass": mass, "empty": empty}


def _evict(name, code, layers, seqs, kv_min, kv_max, budget, recent, hkv, d):
    return {"name": name, "op": "evict", "code": code, "layers": layers, "seqs": seqs,
            "kv_min": kv_min, "kv_max": kv_max, "budget": budget, "recent": recent, "hkv": hkv,
            "d": d}


def listed():
    return [
        # one new token for each of a few short requests on a small model: latency
        _append("append_decode_5", "int8", 5, 1, 37, 611, 2, 64),
        # a decode step of a full serving batch (64 requests, GQA 32/8)
        _append("append_decode_64", "fp8", 64, 1, 129, 2304, 8, 128),
        # continued prefill of four prompts; the chunks begin and end inside a block
        _append("append_chunk_4x2048", "int8", 4, 2048, 2055, 4101, 8, 128),
        # one request on the 14/2-head model: latency
        _attend("decode_1", "int8", 1, 1, 301, 301, 14, 2, 64),
        # the serving benchmark's decode step, its batch padded to 64 rows
        _attend("decode_64", "int8", 64, 1, 129, 2304, 32, 8, 128, empty=3),
        # few long documents: work split along the cache
        _attend("decode_long", "fp8", 3, 1, 20011, 65533, 32, 8, 128),
        # a decode step that also accumulates each cached token's attention weight
        _attend("decode_mass", "int8", 32, 1, 1023, 4096, 32, 8, 128, mass=True),
        # speculative decoding: five drafted tokens verified for each request
        _attend("verify_5", "fp8", 16, 5, 260, 2304, 16, 4, 128),
        # continued prefill: a prompt chunk over the tokens cached before it
        _attend("chunk_1024", "int8", 2, 1024, 3077, 5120, 32, 8, 128),
        # the same while the weights for a later eviction are accumulated
        _attend("chunk_mass", "int8", 2, 511, 1111, 2048, 14, 2, 64, mass=True),
        # one short request of a small model leaves half of its cache
        _evict("evict_1", "int8", 6, 1, 1001, 1001, 500, 64, 2, 64),
        # eight requests of a 32-layer model cut to half of their cache
        _evict("evict_8x32", "fp8", 32, 8, 1500, 4096, 2048, 256, 8, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    code = rng.choice(["int8", "fp8"])
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    op = rng.choice(["append", "attend", "attend", "attend", "evict"])
    if op == "append":
        q = rng.choice([1, 1, _log(rng, 2, 2048)])
        seqs = _log(rng, 1, 64 if q == 1 else 4)
        kv_max = q + _log(rng, 1, 3000)
        c = _append("", code, seqs, q, q + rng.randint(0, kv_max - q), kv_max, hkv, d)
    elif op == "attend":
        group = rng.choice([1, 2, 4, 7, 8])
        kind = rng.choice(["decode", "decode", "verify", "chunk"])
        mass = rng.random() < 0.35
        if kind == "chunk":
            q, seqs = _log(rng, 16, 1024), rng.randint(1, 2)
            group = min(group, 32 // hkv)
            kv_max = q + _log(rng, 1, 4096)
        else:
            q = 1 if kind == "decode" else rng.randint(2, 8)
            seqs = _log(rng, 1, 64)
            kv_max = q + _log(rng, 1, 131072 // seqs)
        empty = rng.randint(0, min(2, seqs - 1))
        c = _attend("", code, seqs, q, q + rng.randint(0, kv_max - q), kv_max, hkv * group, hkv, d,
                    mass, empty)
    else:
        layers, seqs = _log(rng, 1, 24), _log(rng, 1, 8)
        kv_max = _log(rng, 40, 4096)
        budget = rng.randint(max(1, kv_max // 4), max(2, (kv_max * 3) // 4))
        budget = min(budget, 2048)
        c = _evict("", code, layers, seqs, rng.randint(kv_max // 2, kv_max), kv_max, budget,
                   rng.randint(0, budget // 2), hkv, d)
    del c["name"]
    return c


# ------------------------------------------------------------------ the inputs
def _lens(case):
    """Cached lengths, spread evenly between the case's bounds; trailing rows may be empty."""
    n = case["seqs"]
    lens = [case["kv_max"] if n == 1 else
            case["kv_min"] + (case["kv_max"] - case["kv_min"]) * i // (n - 1) for i in range(n)]
    for i in range(case.get("empty", 0)):
        lens[n - 1 - 2 * i] = 0
    return lens


def _pages_of(n):
    return -(-n // PAGE)


def _table(lens, first, order):
    """Page table of sequences of ``lens`` tokens whose pages are order[first], order[first + 1], ..."""
    width = max(1, max(_pages_of(n) for n in lens))
    t = torch.zeros(len(lens), width, dtype=torch.int32)
    for i, n in enumerate(lens):
        k = _pages_of(n)
        t[i, :k] = order[first:first + k]
        first += k
    return t, first


def _fill(codes, scales, code, gen):
    """Quantised keys and values, a few pages at a time: keys have channels of larger
    magnitude, as projections with rotary positions do; values are even."""
    p, h, _, _, d = codes.shape
    chan = torch.ones(2, 1, d, device="cuda")
    big = torch.randperm(d, generator=gen, device="cuda")[:d // 16]
    chan[0, 0, big] = 4.0
    step = max(1, (1 << 26) // (h * 2 * PAGE * d))
    for a in range(0, p, step):
        x = torch.randn(min(step, p - a), h, 2, PAGE, d, generator=gen, device="cuda") * chan
        s = x.abs().amax((-1, -2)) / LEVELS[code]
        scales[a:a + step] = s
        x /= s[..., None, None]
        codes[a:a + step] = (x.round() if code == "int8" else x).to(codes.dtype)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    lens = _lens(case)
    n, hkv, d, code = len(lens), case["hkv"], case["d"], case["code"]
    layers = case.get("layers", 1)
    pages = sum(_pages_of(x) for x in lens)
    kept = [min(x, case.get("budget", 0)) for x in lens]
    total = pages + sum(_pages_of(x) for x in kept) + 1
    order = torch.randperm(total, generator=host).to(torch.int32)
    table, nxt = _table(lens, 0, order)
    codes = torch.zeros(layers, total, hkv, 2, PAGE, d, dtype=STORE[code], device="cuda")
    scales = torch.zeros(layers, total, hkv, 2, device="cuda")
    st = {"case": dict(case), "codes": codes, "scales": scales, "lens_host": lens,
          "table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    for i in range(layers):
        _fill(codes[i], scales[i], code, gen)
    if case["op"] == "evict":
        # attention weight gathers on few tokens; some never received any
        m = torch.rand(layers, total, hkv, PAGE, generator=gen, device="cuda").pow(6) * 40
        st["mass"] = torch.where(m < 1e-6, torch.zeros_like(m), m)
        dst, _ = _table(kept, nxt, order)
        st["dst"] = dst.cuda()
        st["kept"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
        st["kept_host"] = kept
        return st
    q = case["q"]
    st["codes"], st["scales"] = codes[0], scales[0]
    st["cu"] = torch.arange(0, n * q + 1, q, dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        k = torch.randn(n * q, hkv, d, generator=gen, device="cuda")
        k[..., torch.randperm(d, generator=gen, device="cuda")[:d // 16]] *= 4
        st["k"] = k.bfloat16()
        st["v"] = torch.randn(n * q, hkv, d, generator=gen, device="cuda").bfloat16()
        # the pages that the new tokens land on, and how many tokens those then hold
        first = [(x - q) // PAGE for x in lens]
        width = max(_pages_of(x) - f for x, f in zip(lens, first))
        tail = torch.zeros(n, width, dtype=torch.int32)
        for i, (x, f) in enumerate(zip(lens, first)):
            tail[i, :_pages_of(x) - f] = table[i, f:_pages_of(x)]
        st["tail"] = tail.cuda()
        st["tail_lens"] = torch.tensor([x - f * PAGE for x, f in zip(lens, first)],
                                       dtype=torch.int32, device="cuda")
        return st
    st["q"] = (1.5 * torch.randn(n * q, case["hq"], d, generator=gen, device="cuda")).bfloat16()
    st["scale"] = d ** -0.5
    if case["mass"]:
        # weights gathered over the steps before this one
        st["mass"] = torch.rand(total, hkv, PAGE, generator=gen, device="cuda").pow(4) * 8 * q
        st["mass_out"] = st["mass"].clone()
    return st


# ------------------------------------------------------------ the plain forms
def _round(x, code):
    return x.round().clamp(-127, 127).to(torch.int8) if code == "int8" else x.to(STORE[code])


def _gather(codes, scales, table):
    """Keys and values [S, Hkv, pages * 16, D] of a page table, in 32 bits."""
    t = table.long()
    x = codes[t].float() * scales[t][..., None, None]          # [S, pages, Hkv, 2, 16, D]
    s, p, h, _, _, d = x.shape
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, s, h, p * PAGE, d)
    return x[0], x[1]


def _values(codes, scales, table, lens):
    """What the cache holds for these pages, in the model's type; nothing past each length."""
    live = torch.arange(table.shape[1] * PAGE, device="cuda") < lens[:, None]
    return [torch.where(live[:, None, :, None], x, torch.zeros_like(x)).bfloat16()
            for x in _gather(codes, scales, table)]


def _plain_append(st):
    case, codes, scales = st["case"], st["codes"], st["scales"]
    code, q, hkv, d = case["code"], case["q"], case["hkv"], case["d"]
    tail, n = st["tail"].long(), st["tail"].shape[0]
    width = tail.shape[1]
    live = torch.arange(width * PAGE, device="cuda") < st["tail_lens"][:, None]
    start = st["tail_lens"] - q                                 # older tokens of the first block
    slot = start[:, None] + torch.arange(q, device="cuda")      # [S, q]
    new = torch.zeros(n, width * PAGE, hkv, 2, d, device="cuda")
    kv = torch.stack((st["k"].float(), st["v"].float()), 2).view(n, q, hkv, 2, d)
    new[torch.arange(n, device="cuda")[:, None], slot] = kv
    new = new.view(n, width, PAGE, hkv, 2, d).permute(0, 1, 3, 4, 2, 5)
    at = torch.arange(width * PAGE, device="cuda")
    fresh = ((at >= start[:, None]) & live).view(n, width, 1, 1, PAGE, 1)
    held = ((at < start[:, None]) & live).view(n, width, 1, 1, PAGE, 1)
    old_scale = torch.where(held.any(4), scales[tail][..., None], torch.zeros((), device="cuda"))
    levels = torch.full((), LEVELS[code], device="cuda")
    top = new.abs().amax((-1, -2)) / levels
    s = torch.maximum(old_scale[..., 0], top)
    div = torch.where(s > 0, s, torch.ones_like(s))[..., None, None]
    old = codes[tail].float()
    x = torch.where(fresh, new / div, torch.where(held, old * old_scale[..., None] / div, old))
    used = live.view(n, width, PAGE).any(-1)
    pages = tail[used]
    codes[pages] = _round(x, code)[used]
    scales[pages] = s[used]
    k, v = _values(codes, scales, st["tail"], st["tail_lens"])
    return {"k": k, "v": v, "scales": scales}


def _plain_attend(st):
    case = st["case"]
    q_len, hkv, d = case["q"], case["hkv"], case["d"]
    n, group = case["seqs"], case["hq"] // case["hkv"]
    k, v = _gather(st["codes"], st["scales"], st["table"])
    q = st["q"].float().view(n, q_len, hkv, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(n, hkv, group * q_len, d)
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(st["scale"])
    s = s.view(n, hkv, group, q_len, -1)
    pos = st["lens"][:, None] - q_len + torch.arange(q_len, device="cuda")
    seen = torch.arange(s.shape[-1], device="cuda") <= pos[..., None]
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    den = p.sum(-1, keepdim=True)
    p /= torch.where(den > 0, den, torch.ones_like(den))
    o = torch.matmul(p.view(n, hkv, group * q_len, -1), v).view(n, hkv, group, q_len, d)
    out = {"out": o.permute(0, 3, 1, 2, 4).reshape(n * q_len, case["hq"], d).bfloat16()}
    if case["mass"]:
        w = p.sum((2, 3)).view(n, hkv, -1, PAGE).transpose(1, 2)     # [S, pages, Hkv, 16]
        used = torch.arange(st["table"].shape[1], device="cuda") * PAGE < st["lens"][:, None]
        pages = st["table"].long()[used]
        mass = st["mass_out"]
        mass[pages] = st["mass"][pages] + w[used]
        out["mass"] = mass
    return out


def _plain_evict(st):
    case = st["case"]
    code, budget, recent, hkv, d = (case[k] for k in ("code", "budget", "recent", "hkv", "d"))
    layers, n = case["layers"], case["seqs"]
    table, lens, dst = st["table"].long(), st["lens"], st["dst"].long()
    width = table.shape[1] * PAGE
    m = st["mass"][:, table].transpose(2, 3).reshape(layers, n, hkv, width)
    at = torch.arange(width, device="cuda")
    whole = (lens <= budget)[:, None]
    last = (at >= (lens - recent)[:, None]) & (at < lens[:, None])
    rank = torch.where((last | whole)[:, None], float("inf"), m)
    rank = torch.where((at < lens[:, None])[:, None], rank, -1.0)
    rank = torch.nn.functional.pad(rank, (0, max(0, budget - width)), value=-1.0)
    keep = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    slot = torch.arange(budget, device="cuda")
    live = (slot < st["kept"][:, None])[:, None]                       # [S, 1, budget]
    keep = torch.where(live, keep, rank.shape[-1]).sort(-1).values
    src = torch.where(live, keep, 0)
    page = table[torch.arange(n, device="cuda")[:, None, None], src // PAGE]   # [L, S, Hkv, budget]
    lay = torch.arange(layers, device="cuda")[:, None, None, None]
    head = torch.arange(hkv, device="cuda")[:, None]
    pad = dst.shape[1] * PAGE - budget
    old = st["scales"][lay, page, head]                                # [L, S, Hkv, budget, 2]
    old = torch.where(live[..., None], old, torch.zeros_like(old))
    mass = torch.where(live, st["mass"][lay, page, head, src % PAGE], torch.zeros((), device="cuda"))
    x = st["codes"][lay, page, head, :, src % PAGE].float() * old[..., None]
    if pad > 0:
        old = torch.nn.functional.pad(old, (0, 0, 0, pad))
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad))
        mass = torch.nn.functional.pad(mass, (0, pad))
    blocks = dst.shape[1]
    old, x = old[..., :blocks * PAGE, :], x[..., :blocks * PAGE, :, :]
    s = old.view(layers, n, hkv, blocks, PAGE, 2).amax(4)
    div = torch.where(s > 0, s, torch.ones_like(s))
    x = x.view(layers, n, hkv, blocks, PAGE, 2, d) / div[..., None, :, None]
    x = _round(x, code).permute(0, 1, 3, 2, 5, 4, 6)                   # [L, S, blocks, Hkv, 2, 16, D]
    used = torch.arange(blocks, device="cuda") * PAGE < st["kept"][:, None]
    pages = dst[used]
    st["codes"][:, pages] = x[:, used]
    st["scales"][:, pages] = s.permute(0, 1, 3, 2, 4)[:, used]
    mass = mass[..., :blocks * PAGE].view(layers, n, hkv, blocks, PAGE).transpose(2, 3)
    st["mass"][:, pages] = mass[:, used]
    keep = torch.where(live, keep, -1).int()
    k, v = [torch.stack(y) for y in zip(*(_values(st["codes"][i], st["scales"][i], st["dst"], st["kept"])
                                          for i in range(layers)))]
    return {"keep": keep, "k": k, "v": v, "scales": st["scales"], "mass": st["mass"]}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[op](state)
    from complexity_framework_b200.ops import paged8

    if op == "append":
        paged8.paged8_append(state["k"], state["v"], state["codes"], state["scales"],
                             state["table"], state["cu"], state["lens"],
                             max_q_len=state["case"]["q"])
        k, v = paged8.paged8_read(state["codes"], state["scales"], state["tail"],
                                  state["tail_lens"])
        return {"k": k, "v": v, "scales": state["scales"]}
    if op == "attend":
        o = paged8.paged8_attention(state["q"], state["codes"], state["scales"], state["table"],
                                    state["cu"], state["lens"], scale=state["scale"],
                                    max_q_len=state["case"]["q"], mass=state.get("mass"),
                                    mass_out=state.get("mass_out"))
        return {"out": o, "mass": state["mass_out"]} if state["case"]["mass"] else {"out": o}
    keep = paged8.paged8_evict(state["codes"], state["scales"], state["mass"], state["table"],
                               state["lens"], state["dst"], budget=state["case"]["budget"],
                               recent=state["case"]["recent"])
    k, v = paged8.paged8_read(state["codes"], state["scales"], state["dst"], state["kept"])
    return {"keep": keep, "k": k, "v": v, "scales": state["scales"], "mass": state["mass"]}


# ---------------------------------------------------- what a pass cannot avoid
def work(case):
    lens, hkv, d = _lens(case), case["hkv"], case["d"]
    live = sum(lens)
    if case["op"] == "append":
        q = case["q"]
        new = case["seqs"] * q
        held = sum((x - q) % PAGE + q for x in lens)      # tokens of the blocks that are read back
        blocks = sum(_pages_of(x) - (x - q) // PAGE for x in lens)
        return {"bytes": hkv * (new * 2 * d * (2 + 1) + held * 2 * d * 2 + blocks * 2 * 4 * 2),
                "flops": 4 * new * hkv * d}
    if case["op"] == "attend":
        q, hq = case["q"], case["hq"]
        seen = sum(sum(x - q + 1 + i for i in range(q)) for x in lens if x)
        b = live * hkv * 2 * d + sum(_pages_of(x) for x in lens) * (hkv * 2 * 4 + 4) \
            + 2 * case["seqs"] * q * hq * d * 2
        if case["mass"]:
            b += 2 * live * hkv * 4
        return {"bytes": b, "flops": 4 * d * hq * seen}
    kept = sum(min(x, case["budget"]) for x in lens)
    per = case["layers"] * hkv
    blocks = sum(_pages_of(min(x, case["budget"])) for x in lens)
    return {"bytes": per * (live * 4 + kept * (2 * d * 2 + 4 + 4) + kept * 2 * d * 2
                            + 2 * blocks * 2 * 4), "flops": per * kept * 2 * d * 2}


# ----------------------------------------------------- the definition, 64 bits
def _nearest(x, code):
    """The 8-bit number nearest to each value (ties to even), as a 64-bit value."""
    if code == "int8":
        return torch.round(x).clamp(-127, 127)
    a = x.abs().clamp_min(2.0 ** -20)
    ulp = torch.exp2((torch.floor(torch.log2(a)) - 3).clamp_min(-9.0))   # 3 bits below the leading one
    return torch.round(x / ulp).mul(ulp).clamp(-448, 448)


def _sequence(st, i, upto, layer=None):
    """Sequence i's values [2, Hkv, upto, D] in 64 bits."""
    codes = st["codes"] if layer is None else st["codes"][layer]
    scales = st["scales"] if layer is None else st["scales"][layer]
    pages = st["table"][i, :_pages_of(upto)].long()
    if codes.dtype == torch.int8:
        x = codes[pages].double()
    else:
        x = codes[pages].float().double()
    x = x * scales[pages].double()[..., None, None]
    return x.permute(2, 1, 0, 3, 4).flatten(2, 3)[:, :, :upto]


def _exact_append(case, st):
    q, levels = case["q"], LEVELS[case["code"]]
    width = st["tail"].shape[1]
    scales = st["scales"].double()
    res = torch.zeros(2, case["seqs"], case["hkv"], width * PAGE, case["d"], dtype=torch.float64,
                      device="cuda")
    for i, n in enumerate(st["lens_host"]):
        new = torch.stack((st["k"][i * q:(i + 1) * q], st["v"][i * q:(i + 1) * q])).double()
        new = new.transpose(1, 2)                                      # [2, Hkv, q, D]
        start = n - q
        b = start // PAGE
        while b * PAGE < n:
            page = int(st["table"][i, b])
            lo, hi = max(start, b * PAGE), min(n, (b + 1) * PAGE)
            x = new[:, :, lo - start:hi - start]
            s = x.abs().amax((-1, -2)).transpose(0, 1) / levels        # [Hkv, 2]
            at = (b - start // PAGE) * PAGE
            older = lo - b * PAGE
            if older:
                before = scales[page].clone()
                s = torch.maximum(s, before)
                y = st["codes"][page].to(torch.float32).double()[:, :, :older] * before[..., None, None]
                y = _nearest(y / s[..., None, None], case["code"]) * s[..., None, None]
                res[:, i, :, at:at + older] = y.transpose(0, 1)
            st_ = s.transpose(0, 1)[..., None, None]
            res[:, i, :, at + older:at + hi - b * PAGE] = _nearest(x / st_, case["code"]) * st_
            scales[page] = s
            b += 1
    return {"k": res[0], "v": res[1], "scales": scales}


def _exact_attend(case, st):
    q_len, group = case["q"], case["hq"] // case["hkv"]
    out = torch.zeros(case["seqs"], q_len, case["hkv"], group, case["d"], dtype=torch.float64,
                      device="cuda")
    mass = st["mass_out"].double() if case["mass"] else None
    for i, n in enumerate(st["lens_host"]):
        if not n:
            continue
        kv = _sequence(st, i, n)
        add = torch.zeros(case["hkv"], _pages_of(n) * PAGE, dtype=torch.float64, device="cuda")
        hidden = torch.arange(n, device="cuda") > (n - q_len + torch.arange(q_len, device="cuda"))[:, None]
        for h in range(case["hq"]):
            x = st["q"][i * q_len:(i + 1) * q_len, h].double()
            w = (x @ kv[0, h // group].T) * st["scale"]
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[i, :, h // group, h % group] = w @ kv[1, h // group]
            add[h // group, :n] += w.sum(0)
        if case["mass"]:
            pages = st["table"][i, :_pages_of(n)].long()
            mass[pages] += add.view(case["hkv"], -1, PAGE).transpose(0, 1)
    res = {"out": out.reshape(-1, case["hq"], case["d"])}
    return {**res, "mass": mass} if case["mass"] else res


def _exact_evict(case, st):
    budget, recent, hkv = case["budget"], case["recent"], case["hkv"]
    scales, mass = st["scales"].double(), st["mass"].double()
    width = st["dst"].shape[1]
    res = torch.zeros(2, case["layers"], case["seqs"], hkv, width * PAGE, case["d"],
                      dtype=torch.float64, device="cuda")
    for lay in range(case["layers"]):
        for i, n in enumerate(st["lens_host"]):
            pages = st["table"][i, :_pages_of(n)].long()
            m = st["mass"][lay, pages].transpose(0, 1).reshape(hkv, -1)[:, :n]
            if n <= budget:
                idx = torch.arange(n, device="cuda").expand(hkv, n)
            else:
                top = torch.argsort(m[:, :n - recent], dim=-1, descending=True, stable=True)
                idx = torch.cat((top[:, :budget - recent].sort(-1).values,
                                 torch.arange(n - recent, n, device="cuda").expand(hkv, recent)), -1)
            kept = idx.shape[1]
            room = _pages_of(kept) * PAGE
            x = _sequence(st, i, n, lay)                                # [2, Hkv, n, D]
            x = torch.gather(x, 2, idx[None, ..., None].expand(2, -1, -1, case["d"]))
            s = st["scales"][lay, pages].double().permute(2, 1, 0)      # [2, Hkv, pages]
            s = torch.gather(s, 2, (idx // PAGE)[None].expand(2, -1, -1))
            fill = (0, room - kept)
            s = torch.nn.functional.pad(s, fill).view(2, hkv, -1, PAGE).amax(-1)
            wide = s.repeat_interleave(PAGE, -1)[..., :kept, None]
            res[:, lay, i, :, :kept] = _nearest(x / wide, case["code"]) * wide
            to = st["dst"][i, :_pages_of(kept)].long()
            scales[lay, to] = s.permute(2, 1, 0)
            got = torch.nn.functional.pad(torch.gather(m, 1, idx).double(), fill)
            mass[lay, to] = got.view(hkv, -1, PAGE).transpose(0, 1)
    return {"keep": None, "k": res[0], "v": res[1], "scales": scales, "mass": mass}


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](case, st)
