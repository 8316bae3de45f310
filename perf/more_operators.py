"""Operators of a serving loop over a paged KV cache, as cases to time and to compare.

* write: the k and v of new tokens stored into pages, as f16 or quantised to 8 bits (blocks
  of 32 with an f16 scale, as Q8_0), and read back as the values they stand for;
* read: the slots of a sequence read out of its pages, as f32 or f16 rows;
* decode: the attention of one new token of each sequence over its pages, lengths ragged;
* verify: drafted tokens accepted or refused against the target's probabilities from given
  random numbers, and the token after the last accepted one drawn.

With `own` false the same results come from elementary torch operations in f32 (quotients
next to a rounding border and probabilities in f64). Head counts and sizes are those of
bench.py (the 7B and 70B Llama shapes) and of tests/ or generic.

A page holds page slots of every kv head, in units of 32 slots of one head: [page][kv
head][unit]. With nb = ceil(hd / 32) and elements behind hd as zeros, a unit is, for K,
f16 [t 2][b nb][g 4][h 4][j 4][e 8]: slot 8 h + 4 t + j, element 32 b + 8 g + e
q8  int8 [b nb][g 4][h 4][j 4][t 2][e 8], then f16 scales [b nb][slot 32]
and for V
f16 [b nb][t 2][g 4][r 16][e 8]: slot 8 g + e, element 32 b + 16 t + r
q8  int8 [b nb][g 4][r 16][t 2][e 8], then f16 scales [b nb][slot 32].
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
# scores of real heads spread over several units: q of this size against k of about N(0, 1)
Q_SCALE = 3.0
F16, Q8_0, F32 = 1, 8, 0  # GGUF type ids


def listed():
    return [
        # a decode step of 32 sequences: one token each into an 8-bit cache, latency
        {"name": "write_step", "kind": "write", "type": "q8", "seqs": 32, "each": 1, "past": 1500, "kv_heads": 8,
         "hd": 128, "page": 64},
        # a prompt of 4096 tokens into an 8-bit cache
        {"name": "write_prompt", "kind": "write", "type": "q8", "seqs": 1, "each": 4096, "past": 0, "kv_heads": 8,
         "hd": 128, "page": 64},
        # chunks of odd length behind contexts of odd length, f16, heads of 80
        {"name": "write_odd", "kind": "write", "type": "f16", "seqs": 3, "each": 259, "past": 131, "kv_heads": 10,
         "hd": 80, "page": 32},
        # a cached prefix of the 70B context, for the attention of the next chunk of its prompt
        {"name": "read_prefix", "kind": "read", "type": "q8", "seqs": 1, "each": 8192, "past": 0, "kv_heads": 8,
         "hd": 128, "page": 256, "out": "f16"},
        # a short prefix of several sequences, f16 pages, heads of 96
        {"name": "read_short", "kind": "read", "type": "f16", "seqs": 5, "each": 133, "past": 77, "kv_heads": 8,
         "hd": 96, "page": 32, "out": "f32"},
        # one sequence of a 7B shape at the context of bench.py: latency
        {"name": "decode_one", "kind": "decode", "type": "q8", "seqs": 1, "longest": 2048, "heads": 32, "kv_heads": 8,
         "hd": 128, "page": 64},
        # eight sequences of the 70B shape, f16 pages, contexts of all lengths
        {"name": "decode_8", "kind": "decode", "type": "f16", "seqs": 8, "longest": 8191, "heads": 64, "kv_heads": 8,
         "hd": 128, "page": 64},
        # a full batch over an 8-bit cache: the bandwidth bound
        {"name": "decode_64", "kind": "decode", "type": "q8", "seqs": 64, "longest": 8192, "heads": 32, "kv_heads": 8,
         "hd": 128, "page": 128},
        # one q head per kv head, heads of 96, few sequences of odd lengths
        {"name": "decode_odd", "kind": "decode", "type": "f16", "seqs": 5, "longest": 1777, "heads": 12, "kv_heads": 12,
         "hd": 96, "page": 32},
        # four drafted tokens of one sequence: latency
        {"name": "verify_one", "kind": "verify", "seqs": 1, "n": 4, "vocab": 32000, "temp": 0.8, "draft": True},
        # a full batch of long drafts over a large vocabulary
        {"name": "verify_32", "kind": "verify", "seqs": 32, "n": 7, "vocab": 131072, "temp": 1.0, "draft": True},
        # greedy drafts from an n-gram table (no draft probabilities), an odd vocabulary
        {"name": "verify_lookup", "kind": "verify", "seqs": 8, "n": 5, "vocab": 50001, "temp": 0.6, "draft": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "decode", "verify", "verify"])
    if kind == "verify":
        c = {"kind": kind, "seqs": _log(rng, 1, 32), "n": _log(rng, 1, 16), "vocab": _log(rng, 512, 131072),
             "temp": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), "draft": rng.random() < 0.6}
        while c["seqs"] * c["n"] * c["vocab"] > 32 * 7 * 131072:
            c["seqs"] = max(1, c["seqs"] // 2)
            c["n"] = max(1, c["n"] - 2)
        return c
    c = {"kind": kind, "type": rng.choice(["f16", "q8", "q8"]), "kv_heads": rng.choice([1, 2, 4, 8, 10]),
         "hd": rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256]), "page": rng.choice([32, 32, 64, 128, 256])}
    if kind == "decode":
        c.update(seqs=_log(rng, 1, 64), longest=_log(rng, 1, 8192), heads=c["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8, 12, 16]))
        while c["seqs"] * c["longest"] * c["hd"] * max(2 * c["kv_heads"], c["heads"]) > 64 * 8192 * 32 * 128 // 2:
            c["seqs"], c["longest"] = max(1, c["seqs"] // 2), max(1, c["longest"] * 3 // 4)
        return c
    c.update(seqs=_log(rng, 1, 32), past=rng.choice([0, _log(rng, 1, 2000)]))
    c["each"] = _log(rng, 1, 4096 // c["seqs"]) if kind == "write" else _log(rng, 1, 8192 // c["seqs"])
    if kind == "read":
        c["out"] = rng.choice(["f16", "f32"])
    return c


# ---- inputs -----------------------------------------------------------------------------

def _nb(case):
    return (case["hd"] + 31) // 32


def _unit(case):
    """Bytes of 32 slots of one kv head, of K or of V."""
    return _nb(case) * (2048 if case["type"] == "f16" else 1088)


def _pool(case, n_pages, g):
    """A pool of pages as earlier tokens left them: (n_pages, kv heads, units, bytes of a unit)."""
    nb, shape = _nb(case), (n_pages, case["kv_heads"], case["page"] // 32)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float16)  # noqa: E731
    if case["type"] == "f16":
        return randn(*shape, nb * 1024).view(torch.uint8)
    pool = torch.empty(*shape, _unit(case), device=DEV, dtype=torch.uint8)
    pool[..., :nb * 1024] = (randn(*shape, nb * 1024) * 45).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    # blocks of a head differ in size (channels that stand out); about N(0, 1) in all
    size = torch.exp(0.4 * randn(1, case["kv_heads"], 1, nb, 1)) * torch.exp(0.2 * randn(*shape, nb, 32)) * 0.018
    pool[..., nb * 1024:] = size.reshape(*shape, nb * 32).contiguous().view(torch.uint8)
    return pool


def _lens(case):
    """Contexts of all lengths, the longest among them and an odd one."""
    r = random.Random(case["longest"] * 65 + case["seqs"])
    return [case["longest"]] + [r.randint(max(1, case["longest"] // 8), case["longest"]) for _ in range(case["seqs"] - 1)]


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    if case["kind"] == "verify":
        b, n, v = case["seqs"], case["n"], case["vocab"]
        s = {"logits": 2.5 * randn(b, n + 1, v), "u": torch.rand(b, n + 1, generator=g, device=DEV), "draft": None}
        # a draft that mostly agrees; tokens drawn from it (here by noise of the right kind), and some short drafts
        near = s["logits"][:, :n] + 0.5 * randn(b, n, v)
        noise = -torch.log(-torch.log(torch.rand(b, n, v, generator=g, device=DEV).clamp(1e-7, 1 - 1e-7)))
        s["drafted"] = (near + noise * case["temp"]).argmax(-1).int()
        short = torch.rand(b, 1, generator=g, device=DEV) < 0.2
        s["drafted"] = torch.where(short & (torch.arange(n, device=DEV) >= (n + 1) // 2), -1, s["drafted"]).int()
        if case["draft"]:
            s["draft"] = near
        return s
    seqs, kvh, hd, page = case["seqs"], case["kv_heads"], case["hd"], case["page"]
    total = case["longest"] if case["kind"] == "decode" else case["past"] + case["each"]
    per = (total + page - 1) // page
    n_pages = seqs * per + 3
    s = {"table": torch.randperm(n_pages, generator=g, device=DEV)[:seqs * per].reshape(seqs, per).int()}
    s["k"], s["v"] = _pool(case, n_pages, g), _pool(case, n_pages, g)
    if case["kind"] == "decode":
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
        s["q"] = Q_SCALE * randn(seqs, case["heads"] * hd)
        return s
    s["seq"] = torch.arange(seqs, device=DEV, dtype=torch.int32).repeat_interleave(case["each"])
    s["at"] = case["past"] + torch.arange(case["each"], device=DEV, dtype=torch.int32).repeat(seqs)
    if case["kind"] == "write":
        size = torch.exp(0.5 * randn(kvh * hd))  # channels that stand out
        s["new_k"], s["new_v"] = randn(seqs * case["each"], kvh * hd) * size, randn(seqs * case["each"], kvh * hd)
    return s


_dev = None


def _lib():
    global _dev, _V
    if _dev is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "verum-bespoke-singularity_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import vbs_gfx950 as _V
        d = _V.DeviceLib()
        if not d.init():
            raise RuntimeError(d.error())
        _dev = d
    return _dev


class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def prepare(case, seed):
    s = _State(case=case, **_inputs(case, seed))
    if case["kind"] == "verify":
        s.accepted = torch.zeros(case["seqs"], dtype=torch.int32, device=DEV)
        s.tokens = torch.zeros(case["seqs"], case["n"] + 1, dtype=torch.int32, device=DEV)
    elif case["kind"] == "decode":
        s.out = torch.zeros_like(s.q)
    else:
        kind = torch.float16 if case.get("out") == "f16" else torch.float32
        s.out_k, s.out_v = (torch.zeros(case["seqs"] * case["each"], case["kv_heads"] * case["hd"], dtype=kind, device=DEV)
                            for _ in range(2))
    torch.cuda.synchronize()  # the library's own stream does not wait for torch's
    return s


# ---- the plain forms ----------------------------------------------------------------------

def _to_f16_exactly(x):
    """x in f64 rounded once to f16's values (a cast would round to f32 on the way)."""
    _, e = torch.frexp(x)
    step = ((e.clamp(min=-13).long() - 11 + 1023) << 52).view(torch.float64)  # 2^(e - 11), from its bits
    return (torch.round(x / step) * step).half()


def _quantised(x):
    """x (..., blocks, 32): int8 values and f16 scales (..., blocks)."""
    x = x.double()
    top = x.abs().amax(-1)
    d = _to_f16_exactly(top / torch.full_like(top, 127.0))  # (a number as divisor would be its reciprocal times top)
    q = torch.round(x / torch.where(d == 0, math.inf, d.double()).unsqueeze(-1))
    return q.clamp(-127, 127).to(torch.int8), d


def _units(case, x, which):
    """Rows x (units, 32 slots, kv heads, nb * 32) in the order of a unit: (units, kv heads, ...)."""
    n, kvh, nb = x.shape[0], x.shape[2], _nb(case)
    if which == "k":  # slot (h, t, j), element (b, g, e)
        x = x.reshape(n, 4, 2, 4, kvh, nb, 4, 8)
        return x.permute(0, 4, 2, 5, 6, 1, 3, 7) if case["type"] == "f16" else x.permute(0, 4, 5, 6, 1, 3, 2, 7)
    x = x.reshape(n, 4, 8, kvh, nb, 2, 16)  # slot (g, e), element (b, t, r)
    return x.permute(0, 3, 4, 5, 1, 6, 2) if case["type"] == "f16" else x.permute(0, 3, 4, 1, 6, 5, 2)


def _rows(case, units, which):
    """The other way: units (n, kv heads, bytes) as values (n, 32 slots, kv heads, hd) in f32."""
    n, kvh, nb = units.shape[0], units.shape[1], _nb(case)
    if case["type"] == "f16":
        x = units.view(torch.float16).float()
        x = (x.reshape(n, kvh, 2, nb, 4, 4, 4, 8).permute(0, 5, 2, 6, 1, 3, 4, 7) if which == "k" else
             x.reshape(n, kvh, nb, 2, 4, 16, 8).permute(0, 4, 6, 1, 2, 3, 5))
        return x.reshape(n, 32, kvh, nb * 32)[..., :case["hd"]]
    x = units[..., :nb * 1024].contiguous().view(torch.int8).float()
    d = units[..., nb * 1024:].contiguous().view(torch.float16).float().reshape(n, kvh, nb, 32).permute(0, 3, 1, 2)
    x = (x.reshape(n, kvh, nb, 4, 4, 4, 2, 8).permute(0, 4, 6, 5, 1, 2, 3, 7) if which == "k" else
         x.reshape(n, kvh, nb, 4, 16, 2, 8).permute(0, 3, 6, 1, 2, 5, 4))
    return (x.reshape(n, 32, kvh, nb, 32) * d.unsqueeze(-1)).reshape(n, 32, kvh, nb * 32)[..., :case["hd"]]


def _touched(s):
    """The units that hold a token, as an index into (page, unit), and each token's place in them."""
    c, upp = s.case, s.case["page"] // 32
    first, last = c["past"] // 32, (c["past"] + c["each"] - 1) // 32
    unit = torch.arange(first, last + 1, device=DEV)
    page = s.table[:, unit // upp].long().reshape(-1)
    u = (unit % upp).repeat(c["seqs"])
    slot = s.seq.long() * (last + 1 - first) * 32 + s.at.long() - 32 * first
    return page, u, slot


def _plain_write(s):
    c, (page, u, slot) = s.case, _touched(s)
    kvh, hd, nb = c["kv_heads"], c["hd"], _nb(c)
    for pool, new, which in ((s.k, s.new_k, "k"), (s.v, s.new_v, "v")):
        x = torch.zeros(page.numel() * 32, kvh, nb * 32, device=DEV)
        x[slot, :, :hd] = new.reshape(-1, kvh, hd)
        there = torch.zeros(page.numel() * 32, dtype=torch.bool, device=DEV)
        there[slot] = True
        there = there.reshape(-1, 32, 1, 1).expand(-1, -1, kvh, nb * 32)
        old = pool[page, :, u]
        if c["type"] == "f16":
            was = old.view(torch.float16).reshape(-1)
            put = _units(c, x.half().reshape(-1, 32, kvh, nb * 32), which).reshape(-1)
            pool[page, :, u] = torch.where(_units(c, there, which).reshape(-1), put, was).reshape(page.numel(), kvh, -1).view(torch.uint8)
            continue
        q, d = _quantised(x.reshape(-1, kvh, nb, 32))
        was = old[..., :nb * 1024].contiguous().view(torch.int8).reshape(-1)
        put = _units(c, q.reshape(-1, 32, kvh, nb * 32), which).reshape(-1)
        values = torch.where(_units(c, there, which).reshape(-1), put, was).reshape(page.numel(), kvh, -1)
        was = old[..., nb * 1024:].contiguous().view(torch.float16).reshape(-1, kvh, nb, 32)
        d = torch.where(there[..., ::32].permute(0, 2, 3, 1), d.reshape(-1, 32, kvh, nb).permute(0, 2, 3, 1), was)
        scales = d.reshape(page.numel(), kvh, nb * 32).contiguous().view(torch.uint8)
        pool[page, :, u] = torch.cat([values.view(torch.uint8), scales], -1)
    return _plain_read(s)


def _plain_read(s):
    c, (page, u, slot) = s.case, _touched(s)
    for pool, out, which in ((s.k, s.out_k, "k"), (s.v, s.out_v, "v")):
        out.copy_(_rows(c, pool[page, :, u], which).reshape(-1, c["kv_heads"] * c["hd"])[slot])
    return {"k": s.out_k, "v": s.out_v}


def _plain_decode(s):
    c = s.case
    kvh, hd, seqs, group = c["kv_heads"], c["hd"], c["seqs"], c["heads"] // c["kv_heads"]

    def gathered(pool, which):  # (sequences * kv heads, slots, hd)
        units = pool[s.table.long()].transpose(2, 3).reshape(-1, kvh, pool.shape[-1])
        return _rows(c, units, which).reshape(seqs, -1, kvh, hd).transpose(1, 2).reshape(seqs * kvh, -1, hd)
    q = s.q.reshape(seqs * kvh, group, hd)
    k = gathered(s.k, "k").transpose(1, 2).contiguous()
    score = torch.matmul(q, k).reshape(seqs, kvh, group, -1) * (1.0 / math.sqrt(hd))
    see = torch.arange(score.shape[-1], device=DEV) < s.lens.unsqueeze(1)
    score = torch.where(see[:, None, None], score, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    w = (e / e.sum(-1, keepdim=True)).reshape(seqs * kvh, group, -1)
    s.out.copy_(torch.matmul(w, gathered(s.v, "v")).reshape(seqs, -1))
    return s.out


def _plain_verify(s):
    c, (b, n, v) = s.case, (s.case["seqs"], s.case["n"], s.case["vocab"])

    def probabilities(x):
        x = x.double()
        if not c["temp"]:
            return torch.zeros_like(x).scatter_(-1, x.argmax(-1, keepdim=True), 1.0)
        e = torch.exp((x - x.amax(-1, keepdim=True)) / c["temp"])
        return e / e.sum(-1, keepdim=True)
    p = probabilities(s.logits)
    at = s.drafted.long().clamp(0, v - 1).unsqueeze(-1)
    one_hot = s.draft is None or not c["temp"]
    q = torch.zeros(b, n, v, dtype=torch.float64, device=DEV).scatter_(-1, at, 1.0) if one_hot else probabilities(s.draft)
    there = ((s.drafted >= 0) & (s.drafted < v)).long().cumprod(-1)
    yes = s.u[:, :n].double() * q.gather(-1, at).squeeze(-1) < p[:, :n].gather(-1, at).squeeze(-1)
    accepted = (yes.long() * there).cumprod(-1).sum(-1)
    refused = accepted < there.sum(-1)
    row = torch.arange(b, device=DEV)
    r = p[row, accepted]
    less = (r - q[row, accepted.clamp(max=n - 1)]).clamp(min=0)
    r = torch.where((refused & (less.sum(-1) > 0)).unsqueeze(-1), less, r)
    run_to = r.cumsum(-1)
    after = (run_to > s.u[:, n:].double() * run_to[:, -1:]).long().argmax(-1)
    place = torch.arange(n + 1, device=DEV)
    taken = torch.cat([s.drafted.long(), torch.full((b, 1), -1, device=DEV)], 1)
    s.tokens.copy_(torch.where(place < accepted.unsqueeze(1), taken, torch.where(place == accepted.unsqueeze(1), after.unsqueeze(1), -1)))
    s.accepted.copy_(accepted)
    return {"accepted": s.accepted, "tokens": s.tokens}


# ---- one pass -------------------------------------------------------------------------------

def run(s):
    c = s.case
    if not own:
        return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "verify": _plain_verify}[c["kind"]](s)
    dev = _lib()
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    if c["kind"] == "verify":
        v = c["vocab"]
        dev.verify_draft(ptr(s.logits), v, ptr(s.draft), v, ptr(s.drafted), ptr(s.u), c["seqs"], c["n"], v, c["temp"],
                         ptr(s.accepted), ptr(s.tokens))
        return {"accepted": s.accepted, "tokens": s.tokens}
    pages = _V.Pages(ptr(s.k), ptr(s.v), F16 if c["type"] == "f16" else Q8_0, c["page"], s.k.shape[0], c["kv_heads"],
                     c["hd"], ptr(s.table), c["seqs"], s.table.shape[1])
    if c["kind"] == "decode":
        width = c["heads"] * c["hd"]
        dev.attention_paged(pages, 0, ptr(s.q), width, ptr(s.out), width, 0, ptr(s.lens), c["seqs"], c["longest"],
                            c["heads"], 1.0 / math.sqrt(c["hd"]))
        return s.out
    width, n = c["kv_heads"] * c["hd"], c["seqs"] * c["each"]
    if c["kind"] == "write":
        dev.page_store(pages, 0, ptr(s.new_k), ptr(s.new_v), width, ptr(s.seq), ptr(s.at), n)
    dev.page_load(pages, 0, F16 if c.get("out") == "f16" else F32, ptr(s.out_k), ptr(s.out_v), width, ptr(s.seq),
                  ptr(s.at), n)
    return {"k": s.out_k, "v": s.out_v}


# ---- what a pass needs ----------------------------------------------------------------------

def work(case):
    if case["kind"] == "verify":
        b, n, v = case["seqs"], case["n"], case["vocab"]
        rows = b * (n + 1 + (n if case["draft"] and case["temp"] else 0))
        return {"bytes": 4 * rows * v + 4 * b * (3 * n + 3), "flops": 4 * rows * v}
    kvh, hd = case["kv_heads"], case["hd"]
    slot = 2 * kvh * (2 * hd if case["type"] == "f16" else hd + 2 * _nb(case))  # K and V of a slot in pages
    if case["kind"] == "decode":
        slots, row = sum(_lens(case)), case["heads"] * hd
        return {"bytes": slot * slots + 8 * case["seqs"] * row, "flops": 4 * slots * row}
    n = case["seqs"] * case["each"]
    if case["kind"] == "read":
        return {"bytes": n * (slot + 2 * kvh * hd * (2 if case["out"] == "f16" else 4)), "flops": 0}
    return {"bytes": n * (8 * kvh * hd + 2 * slot + 8 * kvh * hd), "flops": 2 * n * kvh * hd}


# ---- the same in 64 bits ---------------------------------------------------------------------

def _where(case, which, slot, element):
    """The index of (slot, element) within a unit's values, from the layout's definition."""
    nb, t8 = _nb(case), case["type"] == "q8"
    b, g8, e = element // 32, element % 32 // 8, element % 8
    if which == "k":
        lane = g8 * 16 + slot // 8 * 4 + slot % 4
        t = slot % 8 // 4
        return ((b * 64 + lane) * 2 + t) * 8 + e if t8 else ((t * nb + b) * 64 + lane) * 8 + e
    lane, t = slot // 8 * 16 + element % 16, element % 32 // 16
    return ((b * 64 + lane) * 2 + t) * 8 + slot % 8 if t8 else ((b * 2 + t) * 64 + lane) * 8 + slot % 8


def _slots(case, s, which, seq, first, end):
    """Slots first .. end - 1 of a sequence in f64: (slots, kv heads, hd)."""
    j, page = torch.arange(first, end, device=DEV), case["page"]
    pool = s[which]
    units = pool[s["table"][seq].long()[j // page], :, j % page // 32]  # (slots, kv heads, bytes)
    el = torch.arange(case["hd"], device=DEV)
    at = _where(case, which, (j % 32).unsqueeze(1), el.unsqueeze(0)).unsqueeze(1).expand(-1, units.shape[1], -1)
    if case["type"] == "f16":
        return units.view(torch.float16).gather(2, at).to(torch.float64)
    cut = 1024 * _nb(case)
    d = units[..., cut:].contiguous().view(torch.float16).gather(2, (el // 32 * 32 + (j % 32).unsqueeze(1)).unsqueeze(1).expand_as(at))
    return units[..., :cut].contiguous().view(torch.int8).gather(2, at).to(torch.float64) * d.to(torch.float64)


def _held(case, x):
    """What a page holds of rows x (n, kv heads * hd), in f64."""
    if case["type"] == "f16":
        return x.to(torch.float16).to(torch.float64)
    x = x.to(torch.float64).reshape(-1, case["kv_heads"], case["hd"])
    out = torch.empty_like(x)
    for b in range(0, case["hd"], 32):
        part = x[..., b:b + 32]
        d = torch.from_numpy((part.abs().amax(-1, keepdim=True).cpu().numpy() / 127).astype("float16").astype("float64")).to(DEV)
        out[..., b:b + 32] = torch.where(d > 0, torch.round(part / d).clamp(-127, 127) * d, 0.0)
    return out.reshape(x.shape[0], -1)


def exact(case, seed):
    s, f64, kind = _inputs(case, seed), torch.float64, case["kind"]
    if kind == "verify":
        b, n, v = case["seqs"], case["n"], case["vocab"]
        accepted, tokens = torch.zeros(b, dtype=torch.int32), torch.full((b, n + 1), -1, dtype=torch.int32)
        share = lambda row: torch.softmax(row.to(f64) / case["temp"], -1)  # noqa: E731
        for i in range(b):
            k, less = 0, None
            while k < n and int(s["drafted"][i, k]) >= 0:
                x = int(s["drafted"][i, k])
                if not case["temp"]:
                    if int(s["logits"][i, k].argmax()) != x:
                        break
                else:
                    p = share(s["logits"][i, k])
                    if s["draft"] is None:
                        q = torch.zeros_like(p)
                        q[x] = 1.0
                    else:
                        q = share(s["draft"][i, k])
                    if not float(s["u"][i, k]) * float(q[x]) < float(p[x]):
                        less = torch.clamp(p - q, min=0)
                        break
                tokens[i, k] = x
                k += 1
            accepted[i] = k
            if not case["temp"]:
                tokens[i, k] = int(s["logits"][i, k].argmax())
                continue
            r = less if less is not None and float(less.sum()) > 0 else share(s["logits"][i, k])
            c = torch.cumsum(r, 0)
            tokens[i, k] = int(torch.searchsorted(c, float(s["u"][i, n]) * c[-1], right=True))
        return {"accepted": accepted, "tokens": tokens}
    kvh, hd = case["kv_heads"], case["hd"]
    if kind == "write":
        return {"k": _held(case, s["new_k"]), "v": _held(case, s["new_v"])}
    if kind == "read":
        span = (case["past"], case["past"] + case["each"])
        return {w: torch.cat([_slots(case, s, w, i, *span) for i in range(case["seqs"])]).reshape(-1, kvh * hd) for w in "kv"}
    out = torch.empty(case["seqs"], case["heads"], hd, dtype=f64, device=DEV)
    group = case["heads"] // kvh
    for i, length in enumerate(_lens(case)):
        k, v = (_slots(case, s, w, i, 0, length) for w in "kv")
        q = s["q"][i].to(f64).reshape(kvh, group, hd)
        for h in range(kvh):
            w = torch.softmax(q[h] @ k[:, h].T.contiguous() / math.sqrt(hd), -1)
            out[i, h * group:(h + 1) * group] = w @ v[:, h]
    return out.reshape(case["seqs"], -1)
