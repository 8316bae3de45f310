"""Operators for steps of several tokens over the f16 KV cache, as cases to time and to compare.

* rope: rotary positions with several axes (time, height, width) of n tokens, q
  rotated in place, k rotated and k and v stored into the f16 cache;
* tree: the attention of a tree of drafted tokens over the cache;
* chunk: the attention of n consecutive tokens over the cache, with scores capped
  by a tanh, a bias that depends on distance, a document mask or a prefix, and the
  attention weight that each slot received added up (n = 1 is a decode step);
* evict: the cache cut to a budget of slots by that accumulated weight.

With `own` false the same results come from elementary torch operations in f32.
Head counts and sizes are those of bench.py (the 7B and 70B Llama shapes) and of
tests/ or generic.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
# scores of real heads spread over several units: q of this size against k of N(0, 1)
Q_SCALE = 3.0


def listed():
    return [
        # one token of a decode loop with time, height and width positions: latency
        {"name": "rope_token", "kind": "rope", "n": 1, "heads": 32, "kv_heads": 8, "hd": 128, "sections": "16,24,24",
         "slot": 2047, "far": 4096},
        # the patches of an image, and the far positions of a long video
        {"name": "rope_image", "kind": "rope", "n": 1024, "heads": 64, "kv_heads": 8, "hd": 128,
         "sections": "16,24,24", "slot": 1001, "far": 1000000},
        # a small draft of a 7B shape at the context of bench.py
        {"name": "tree_16", "kind": "tree", "n": 16, "past": 2048, "heads": 32, "kv_heads": 8, "hd": 128},
        # a wide draft of the 70B shape over a long context
        {"name": "tree_64_long", "kind": "tree", "n": 64, "past": 8191, "heads": 64, "kv_heads": 8, "hd": 128},
        # odd numbers of tokens and slots, heads of 96
        {"name": "tree_odd", "kind": "tree", "n": 37, "past": 3001, "heads": 32, "kv_heads": 8, "hd": 96},
        # one token with capped scores over the 70B context
        {"name": "decode_cap", "kind": "chunk", "n": 1, "past": 8191, "heads": 64, "kv_heads": 8, "hd": 128,
         "cap": 50.0, "slopes": False, "docs": 0, "prefix": 0, "mass": False},
        # one token of a loop that keeps its cache within a budget: the weights are accumulated
        {"name": "decode_mass", "kind": "chunk", "n": 1, "past": 2047, "heads": 32, "kv_heads": 8, "hd": 128,
         "cap": 0.0, "slopes": False, "docs": 0, "prefix": 0, "mass": True},
        # several short texts packed into one pass, with a distance bias; one q head per kv head of 64
        {"name": "packed_docs", "kind": "chunk", "n": 777, "past": 0, "heads": 16, "kv_heads": 16, "hd": 64,
         "cap": 0.0, "slopes": True, "docs": 200, "prefix": 0, "mass": False},
        # a bidirectional prefix before the text, heads of 80 (no multiple of 32), weights accumulated
        {"name": "prefix_mass", "kind": "chunk", "n": 512, "past": 131, "heads": 10, "kv_heads": 2, "hd": 80,
         "cap": 0.0, "slopes": False, "docs": 0, "prefix": 387, "mass": True},
        # the last chunk of a long prompt, capped: the arithmetic bound
        {"name": "prompt_cap", "kind": "chunk", "n": 2048, "past": 6144, "heads": 32, "kv_heads": 8, "hd": 128,
         "cap": 30.0, "slopes": False, "docs": 0, "prefix": 0, "mass": False},
        # one layer cut to half
        {"name": "evict_layer", "kind": "evict", "layers": 1, "len": 2049, "budget": 1024, "first": 4, "last": 256,
         "kv_heads": 8, "hd": 128},
        # every layer of the 7B shape cut from 8192 slots to 4096
        {"name": "evict_model", "kind": "evict", "layers": 32, "len": 8192, "budget": 4096, "first": 4, "last": 512,
         "kv_heads": 8, "hd": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "tree", "tree", "chunk", "chunk", "chunk", "evict"])
    kvh = rng.choice([1, 2, 4, 8])
    heads = kvh * rng.choice([1, 2, 3, 4, 5, 8])
    hd = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
    if kind == "rope":
        axes = rng.randint(1, 4)
        cuts = sorted(rng.sample(range(1, hd // 2), axes - 1))
        return {"kind": "rope", "n": _log(rng, 1, 4096), "heads": heads, "kv_heads": kvh, "hd": hd,
                "sections": ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [hd // 2])),
                "slot": _log(rng, 1, 3000), "far": _log(rng, 4096, 1000000)}
    if kind == "tree":
        return {"kind": "tree", "n": _log(rng, 1, 160), "past": _log(rng, 1, 16384), "heads": heads, "kv_heads": kvh,
                "hd": hd}
    if kind == "chunk":
        n = _log(rng, 1, 2048)
        past = rng.choice([0, _log(rng, 1, 8192)])
        while n * (past + n) * heads * hd > 2048 * 8192 * 32 * 128 // 2:
            n, past = max(1, n // 2), past // 2
        return {"kind": "chunk", "n": n, "past": past, "heads": heads, "kv_heads": kvh, "hd": hd,
                "cap": rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), "slopes": rng.random() < 0.3,
                "docs": rng.choice([0, 0, _log(rng, 16, 1024)]),
                "prefix": rng.choice([0, 0, rng.randint(1, past + n)]), "mass": rng.random() < 0.3}
    length = _log(rng, 16, 16384)
    hd = min(hd, 128)
    budget = rng.randint(max(1, length // 8), length)
    first = rng.randint(0, min(8, budget))
    return {"kind": "evict", "layers": rng.randint(1, 8), "len": length, "budget": budget, "first": first,
            "last": rng.randint(0, budget - first) // 2, "kv_heads": kvh, "hd": hd}


# ---- inputs -----------------------------------------------------------------------------

THETA = 10000.0
SPARE = 9  # slots of the cache behind the last one in use


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _documents(case):
    """The document of every slot: texts of random lengths around case["docs"], of a fixed draw."""
    total, ids, r = case["past"] + case["n"], [], random.Random(case["docs"])
    while len(ids) < total:
        ids += [ids[-1] + 1 if ids else 0] * max(1, int(case["docs"] * r.uniform(0.3, 1.7)))
    return ids[:total]


def _tree(n, seed):
    """Mask rows of a random tree of n drafted tokens: token i sees its ancestors and itself."""
    r, rows = random.Random(int(seed)), []
    for i in range(n):
        parent = r.randint(-1 if i < 4 else max(0, i - 12), i - 1) if i else -1
        rows.append((rows[parent] if parent >= 0 else 0) | 1 << i)
    words = (n + 63) // 64
    signed = lambda v: v - (1 << 64) if v >> 63 else v  # noqa: E731
    return [[signed(row >> 64 * w & (1 << 64) - 1) for w in range(words)] for row in rows]


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    k = case["kind"]
    randn = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device=DEV, dtype=dtype)  # noqa: E731
    if k == "evict":
        shape = (case["layers"], case["len"] + SPARE, case["kv_heads"] * case["hd"])
        mass = torch.exp(2.5 * randn(case["layers"], case["kv_heads"], shape[1]))
        # slots that no query looked at: equal weights
        mass[torch.rand(mass.shape, generator=g, device=DEV) < 0.05] = 0.0
        return {"kc": randn(*shape, dtype=torch.float16), "vc": randn(*shape, dtype=torch.float16), "mass": mass}
    n, qd, kvd = case["n"], case["heads"] * case["hd"], case["kv_heads"] * case["hd"]
    s = {"q": randn(n, qd)}
    slots = (case["slot"] if k == "rope" else case["past"]) + n + SPARE
    if k == "rope":
        s["k"], s["v"] = randn(n, kvd), randn(n, kvd)
        s["kc"], s["vc"] = (torch.zeros(1, slots, kvd, device=DEV, dtype=torch.float16) for _ in range(2))
        s["pos"] = torch.randint(0, case["far"], (len(_sections(case)), n), generator=g, device=DEV, dtype=torch.int32)
        return s
    s["q"] *= Q_SCALE
    s["kc"], s["vc"] = randn(1, slots, kvd, dtype=torch.float16), randn(1, slots, kvd, dtype=torch.float16)
    s["out"] = torch.zeros(n, qd, device=DEV)
    if k == "tree":
        s["mask"] = torch.tensor(_tree(n, seed), dtype=torch.int64, device=DEV)
        return s
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device=DEV) / case["heads"]).float() if case["slopes"] else None
    s["docs"] = torch.tensor(_documents(case), dtype=torch.int32, device=DEV) if case["docs"] else None
    s["mass"] = torch.rand(1, case["kv_heads"], slots, generator=g, device=DEV) * 4 if case["mass"] else None
    return s


_dev = None


def _lib():
    global _dev
    if _dev is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "verum-bespoke-singularity_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import vbs_gfx950 as V
        d = V.DeviceLib()
        if not d.init():
            raise RuntimeError(d.error())
        _dev = d
    return _dev


class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def prepare(case, seed):
    s = _State(case=case, **_inputs(case, seed))
    if case["kind"] == "evict":
        s.kept = torch.zeros(case["layers"], case["kv_heads"], case["budget"], dtype=torch.int32, device=DEV)
        s.mass_out = torch.zeros_like(s.mass)
    torch.cuda.synchronize()  # the library's own stream does not wait for torch's
    return s


# ---- the plain forms ----------------------------------------------------------------------

def _rotate(x, pos, sections, hd):
    """x (n, heads * hd) rotated in pairs (2p, 2p + 1): angles in 64 bits, their cosines and the products in 32."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device=DEV), torch.tensor(sections, device=DEV))
    freq = THETA ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / -hd)
    angle = pos[axis].T.double() * freq  # (n, pairs)
    c, sn = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    a, b = x.reshape(x.shape[0], -1, hd // 2, 2).unbind(-1)
    return torch.stack([a * c - b * sn, a * sn + b * c], -1).reshape(x.shape)


def _weights(q, k, see, scale, cap=0.0, slopes=None, at=None):
    """Attention weights (kv heads, tokens, group, slots) of q (tokens, heads, hd) over k (slots, kv heads, hd) where `see`
    (tokens, slots); `at` the slots of the tokens."""
    n, heads, hd = q.shape
    slots, kvh, _ = k.shape
    rows = q.reshape(n, kvh, heads // kvh, hd).permute(1, 0, 2, 3).reshape(kvh, -1, hd)
    s = torch.matmul(rows, k.permute(1, 2, 0).contiguous()).reshape(kvh, n, heads // kvh, slots) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        far = (at.unsqueeze(1) - torch.arange(slots, device=DEV)).abs().float()
        s = s - slopes.reshape(kvh, 1, -1, 1) * far.unsqueeze(1)
    s = torch.where(see.unsqueeze(1), s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def _mix(w, v):
    """(tokens, heads * hd) from weights (kv heads, tokens, group, slots) and v (slots, kv heads, hd)."""
    kvh, n, group, slots = w.shape
    out = torch.matmul(w.reshape(kvh, n * group, slots), v.permute(1, 0, 2).contiguous())
    return out.reshape(kvh, n, group, -1).permute(1, 0, 2, 3).reshape(n, -1)


def _plain_attention(s):
    c = s.case
    n, past, kvh, hd = c["n"], c["past"], c["kv_heads"], c["hd"]
    total = past + n
    k, v = (x[0, :total].float().reshape(total, kvh, hd) for x in (s.kc, s.vc))
    q, scale = s.q.reshape(n, -1, hd), 1.0 / math.sqrt(hd)
    slot = torch.arange(total, device=DEV)
    at = past + torch.arange(n, device=DEV)
    if c["kind"] == "tree":
        drafted = torch.arange(n, device=DEV)
        bits = (s.mask[:, drafted // 64] >> (drafted % 64)) & 1
        see = torch.cat([torch.ones(n, past, dtype=torch.bool, device=DEV), bits.bool()], 1)
        s.out.copy_(_mix(_weights(q, k, see, scale), v))
        return s.out
    see = (slot <= at.unsqueeze(1)) | (slot < c["prefix"])
    if s.docs is not None:
        see &= s.docs == s.docs[past:].unsqueeze(1)
    w = _weights(q, k, see, scale, c["cap"], s.slopes, at)
    s.out.copy_(_mix(w, v))
    if s.mass is None:
        return s.out
    s.mass[0, :, :total] += w.sum((1, 2))
    return {"out": s.out, "mass": s.mass}


def _plain_evict(s):
    c = s.case
    length, budget, first, last, hd = c["len"], c["budget"], c["first"], c["last"], c["hd"]
    key = s.mass[:, :, :length].clone()
    key[:, :, :first] = math.inf
    key[:, :, length - last:] = math.inf
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices  # equal weights: the lowest slot first
    kept = torch.sort(order[:, :, :budget], dim=-1).values  # (layers, kv heads, budget)
    s.kept.copy_(kept)
    s.mass_out[:, :, :budget] = torch.gather(s.mass, 2, kept)
    s.mass_out[:, :, budget:length] = 0.0
    rows = kept.permute(0, 2, 1).unsqueeze(-1).expand(-1, -1, -1, hd)
    moved = [torch.gather(x.reshape(*x.shape[:2], -1, hd), 1, rows).reshape(x.shape[0], budget, -1) for x in (s.kc, s.vc)]
    s.kc[:, :budget] = moved[0]
    s.vc[:, :budget] = moved[1]
    return {"k": s.kc, "v": s.vc, "kept": s.kept, "mass": s.mass_out}


def _plain(s):
    c = s.case
    if c["kind"] == "evict":
        return _plain_evict(s)
    if c["kind"] != "rope":
        return _plain_attention(s)
    to = slice(c["slot"], c["slot"] + c["n"])
    s.q.copy_(_rotate(s.q, s.pos, _sections(c), c["hd"]))
    s.kc[0, to] = _rotate(s.k, s.pos, _sections(c), c["hd"]).half()
    s.vc[0, to] = s.v.half()
    return {"q": s.q, "k": s.kc[0, to], "v": s.vc[0, to]}


# ---- one pass -------------------------------------------------------------------------------

def run(s):
    if not own:
        return _plain(s)
    dev, c = _lib(), s.case
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    kvh, hd = c["kv_heads"], c["hd"]
    if c["kind"] == "evict":
        dev.cache_evict(ptr(s.kc), ptr(s.vc), ptr(s.mass), ptr(s.mass_out), ptr(s.kept), c["len"], c["budget"],
                        c["first"], c["last"], 0, c["layers"], s.kc.shape[1], kvh, hd)
        return {"k": s.kc, "v": s.vc, "kept": s.kept, "mass": s.mass_out}
    heads, n, slots = c["heads"], c["n"], s.kc.shape[1]
    if c["kind"] == "rope":
        dev.rope_axes(ptr(s.q), heads * hd, ptr(s.k), ptr(s.v), kvh * hd, ptr(s.pos), n, _sections(c), ptr(s.kc),
                      ptr(s.vc), c["slot"], 0, slots, heads, kvh, hd, THETA)
        to = slice(c["slot"], c["slot"] + n)
        return {"q": s.q, "k": s.kc[0, to], "v": s.vc[0, to]}
    shape = (0, slots, heads, kvh, hd, 1.0 / math.sqrt(hd))
    if c["kind"] == "tree":
        dev.attention_tree(ptr(s.q), heads * hd, ptr(s.kc), ptr(s.vc), ptr(s.out), heads * hd, n, c["past"],
                           ptr(s.mask), *shape)
        return s.out
    dev.attention_chunk(ptr(s.q), heads * hd, ptr(s.kc), ptr(s.vc), ptr(s.out), heads * hd, n, c["past"], *shape,
                        cap=c["cap"], slopes=ptr(s.slopes), docs=ptr(s.docs), prefix=c["prefix"], mass=ptr(s.mass))
    return s.out if s.mass is None else {"out": s.out, "mass": s.mass}


# ---- what a pass needs ----------------------------------------------------------------------

def _seen(case):
    """Pairs of a token and a slot that it sees, summed over the tokens (the drafted part of a tree at a token's depth
    of about log2 n)."""
    n, past = case["n"], case["past"]
    if case["kind"] == "tree":
        return n * past + n * max(1, int(math.log2(n + 1)))
    if not case["docs"]:
        return sum(max(past + i + 1, min(case["prefix"], past + n)) for i in range(n))
    ids = _documents(case)
    start, end = {}, {}
    for j, d in enumerate(ids):
        start.setdefault(d, j)
        end[d] = j + 1
    top = lambda i, d: max(i + 1, min(end[d], case["prefix"]))  # noqa: E731
    return sum(top(i, ids[i]) - start[ids[i]] for i in range(past, past + n))


def work(case):
    k, kvh, hd = case["kind"], case["kv_heads"], case["hd"]
    if k == "evict":
        rows = case["layers"] * kvh * (case["budget"] - case["first"])
        return {"bytes": rows * 8 * hd + case["layers"] * kvh * (8 * case["len"] + 4 * case["budget"]), "flops": 0}
    n, heads = case["n"], case["heads"]
    if k == "rope":
        return {"bytes": n * hd * (8 * heads + 12 * kvh) + 4 * n * len(_sections(case)), "flops": 3 * n * hd * (heads + kvh)}
    total = case["past"] + n
    seen = _seen(case)
    low = 0
    if k == "chunk" and case["docs"]:
        ids = _documents(case)
        low = ids.index(ids[case["past"]])  # slots of earlier documents are not read
    mass = 8 * kvh * (total - low) if k == "chunk" and case["mass"] else 0
    return {"bytes": 4 * kvh * hd * (total - low) + 8 * n * heads * hd + mass, "flops": 4 * hd * heads * seen}


# ---- the same in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s, k, f64 = _inputs(case, seed), case["kind"], torch.float64
    kvh, hd = case["kv_heads"], case["hd"]
    if k == "evict":
        budget, length = case["budget"], case["len"]
        mass = s["mass"].clone()
        for layer in range(case["layers"]):
            for h in range(kvh):
                at = torch.arange(length, device=DEV)
                free = (at >= case["first"]) & (at < length - case["last"])
                middle = at[free]
                # a slot's place: the slots of more weight, then those of the same weight before it
                score = s["mass"][layer, h][middle].to(f64)
                best = middle[torch.argsort(-score, stable=True)[:budget - case["first"] - case["last"]]]
                keep = torch.cat([at[~free], best]).sort().values
                mass[layer, h, :budget] = s["mass"][layer, h][keep]
                for c in ("kc", "vc"):
                    head = s[c][layer, :, h * hd:(h + 1) * hd]
                    head[:budget] = head[keep]
        out = torch.zeros_like(mass)
        out[:, :, :budget] = mass[:, :, :budget]
        return {"k": s["kc"].to(f64), "v": s["vc"].to(f64), "kept": None, "mass": out.to(f64)}
    n, heads = case["n"], case["heads"]
    if k == "rope":
        def turned(x):
            z = torch.view_as_complex(x.to(f64).reshape(n, -1, hd // 2, 2).contiguous())
            parts, p = [], 0
            for axis, width in enumerate(_sections(case)):
                exponent = -2.0 * torch.arange(p, p + width, device=DEV, dtype=f64) / hd
                angle = s["pos"][axis].to(f64)[:, None] * torch.exp(exponent * math.log(THETA))[None]
                parts.append(z[:, :, p:p + width] * torch.polar(torch.ones_like(angle), angle)[:, None])
                p += width
            return torch.view_as_real(torch.cat(parts, -1)).reshape(n, -1)
        return {"q": turned(s["q"]), "k": turned(s["k"]), "v": s["v"].to(f64)}
    past = case["past"]
    total, group = past + n, heads // kvh
    i, j = torch.arange(past, total, device=DEV)[:, None], torch.arange(total, device=DEV)[None]
    if k == "tree":
        hidden = torch.zeros(n, total, dtype=torch.bool, device=DEV)
        for t in range(n):
            hidden[:, past + t] = s["mask"][:, t // 64].bitwise_and(torch.tensor(1, device=DEV) << t % 64) == 0
    else:
        hidden = (j > i) & (j >= case["prefix"])
        if s["docs"] is not None:
            hidden |= s["docs"].to(f64)[None] != s["docs"].to(f64)[past:, None]
    out, got = torch.zeros(n, heads, hd, dtype=f64, device=DEV), []
    q = s["q"].to(f64).reshape(n, heads, hd)
    for h in range(kvh):
        key, value = (s[c][0, :total, h * hd:(h + 1) * hd].to(f64) for c in ("kc", "vc"))
        sums = torch.zeros(total, dtype=f64, device=DEV)
        for a in range(h * group, (h + 1) * group):
            score = q[:, a] @ key.T.contiguous() / math.sqrt(hd)
            if k == "chunk" and case["cap"]:
                score = torch.tanh(score / case["cap"]) * case["cap"]
            if k == "chunk" and case["slopes"]:
                score = score - s["slopes"][a].to(f64) * (i - j).abs()
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            out[:, a] = p @ value
            sums += p.sum(0)
        got.append(sums)
    if k == "tree" or s["mass"] is None:
        return out.reshape(n, -1)
    mass = s["mass"].to(f64)
    mass[0, :, :total] += torch.stack(got)
    return {"out": out.reshape(n, -1), "mass": mass}
