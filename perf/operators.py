"""Long contexts in a cache of 4 bits, and beams over it: the operators, as cases that can be timed and compared.

    listed()              the cases themselves
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   inputs and buffers a program has before the call
    run(state)            one pass: the library's operators where `own` is set, else the same in elementary torch operations
    work(case)            bytes and operations the pass cannot do without
    exact(case, seed)     the outputs in 64 bits, from the definitions

Kinds of cases:
    append    rotary positions, and new keys and values rounded to 4 bits into the cache (lcu_cache4_append); the written rows
              are read back as the values they stand for (lcu_cache4_read)
    attend    attention of prompt rows or single tokens over such a cache (lcu_attention_cache4), with or without the attention
              weight that each cached row received
    evict     the rows of a cache that received the most weight, and its latest ones, are kept (lcu_cache_evict)
    beam      the best continuations of a group of beams and the reordering of their caches (lcu_beam_select, lcu_cache_reorder)

A 4-bit cache holds, per sequence and key/value head, rows of codes and scales.  With absmax the largest magnitude of a block of
`block` neighbouring dimensions, the block's scale is absmax / 7.5 rounded to 7 significant bits, at most 8704, held as a half; the code
of x is floor(x / scale + 8) within 0 .. 15 and stands for (code - 7.5) * scale.  The eight codes of dimensions 32 g + 8 o .. + 7 are
the nibbles, lowest first, of the row's 32-bit word o * (head_dim / 32) + g.
"""
import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
NUMBER = {"f16": 0, "bf16": 1, "f32": 2}


def library():
    if "llama_cu_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("llama_cu_b200", os.path.join(ROOT, "llama.cu_b200", "__init__.py"))
        module = importlib.util.module_from_spec(spec)
        sys.modules["llama_cu_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["llama_cu_b200"]


# ------------------------------------------------------------------ cases
def append(name, seqs, rows, held, heads, kv, dim=128, block=32, dtype="f16", shift=0, theta=10000.0):
    """`held` rows are in each cache already (fewer in later sequences); positions are `shift` ahead of the rows, as behind an eviction."""
    return {"name": name, "kind": "append", "seqs": seqs, "rows": rows, "held": held, "heads": heads, "kv": kv, "dim": dim, "block": block,
            "dtype": dtype, "shift": shift, "theta": theta}


def attend(name, seqs, rows, held, heads, kv, dim=128, block=32, dtype="f16", weights=False):
    return {"name": name, "kind": "attend", "seqs": seqs, "rows": rows, "held": held, "heads": heads, "kv": kv, "dim": dim, "block": block,
            "dtype": dtype, "weights": weights}


def evict(name, seqs, held, keep, recent, kv, dim=128):
    return {"name": name, "kind": "evict", "seqs": seqs, "held": held, "keep": keep, "recent": recent, "kv": kv, "dim": dim}


def beam(name, groups, beams, vocab, held, kv, dim=128, dtype="f16"):
    return {"name": name, "kind": "beam", "groups": groups, "beams": beams, "vocab": vocab, "held": held, "kv": kv, "dim": dim, "dtype": dtype}


def listed():
    return [
        # one token of a 7B-shaped model's layer, interactive: latency
        append("append 1 token", 1, 1, 700, 32, 32),
        # a long document's prompt in one pass, queries of several heads per key head
        append("append 1999 rows bf16", 1, 1999, 0, 32, 8, block=64, dtype="bf16"),
        # the same token's attention over a short conversation
        attend("decode 1 x 32 heads 700", 1, 1, 700, 32, 32),
        # serving: sixteen sequences of long contexts, grouped heads
        attend("decode 16 x 16000 grouped", 16, 1, 15999, 32, 8, block=64, dtype="bf16"),
        # one very long context whose rows' weights decide what is evicted later
        attend("decode 32000 weights", 1, 1, 31999, 32, 32, weights=True),
        # time to the first token of an ordinary prompt
        attend("prompt 509", 1, 509, 0, 32, 32),
        # a question of 2000 tokens behind a cached document, with the weights
        attend("prompt 2000 behind 6000", 1, 2000, 6000, 32, 8, block=64, dtype="bf16", weights=True),
        # a full context of 2048 gives half of its rows up
        evict("evict 2048 to 1024", 1, 2048, 1024, 256, 32),
        # four long contexts, an odd number of rows kept
        evict("evict 4 x 16000 to 8001", 4, 16000, 8001, 333, 8),
        # an ordinary beam search: four beams, the layer's cache behind it
        beam("beam 4 of 32000", 1, 4, 32000, 300, 8),
        # eight requests at once
        beam("beam 8 x 4 of 32000", 8, 4, 32000, 1000, 8, dtype="bf16"),
        # wide beams over a large vocabulary in 32-bit logits
        beam("beam 4 x 16 of 128000", 4, 16, 128000, 500, 4, dtype="f32"),
    ]


def log_int(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "evict", "beam"])
    kv, group, dim = rng.choice([1, 2, 4, 5, 8, 8, 16, 32]), rng.choice([1, 1, 2, 4, 4, 7, 8, 12]), rng.choice([64, 128, 128])
    while kv * group > 64:
        kv //= 2
    block = rng.choice([b for b in (32, 32, 64, 128) if b <= dim])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "append":
        rows = rng.choice([1, log_int(rng, 2, 1999)])
        seqs = log_int(rng, 1, min(16, max(1, 2500 // rows)))
        c = append(None, seqs, rows, log_int(rng, 1, 4000) - 1, kv * group, kv, dim, block, dtype, rng.choice([0, log_int(rng, 1, 100000)]),
                   rng.choice([10000.0, 500000.0]))
    elif kind == "attend":
        rows = rng.choice([1, 1, log_int(rng, 2, 2000)])
        held = log_int(rng, 1, 32000 if rows == 1 else 6000) - 1
        seqs = max(1, min(log_int(rng, 1, 16), 16 * 8 * 16000 * 128 // ((held + rows) * kv * dim)))
        if rows > 1:
            seqs = max(1, min(seqs, 2000 * 7000 * 32 // (rows * (held + rows) * kv * group)))
        c = attend(None, seqs, rows, held, kv * group, kv, dim, block, dtype, rng.random() < 0.4)
    elif kind == "evict":
        held = log_int(rng, 3, 32000)
        keep = rng.randint(max(1, held // 4), held)
        c = evict(None, max(1, min(log_int(rng, 1, 8), 4 * 16000 * 8 * 128 // (held * kv * dim))), held, keep, rng.randint(0, keep // 2), kv, dim)
    else:
        beams, held = rng.choice([1, 2, 3, 4, 4, 8, 16]), log_int(rng, 1, 2000)
        kv = min(kv, 8)
        vocab = log_int(rng, 500, 128000)
        c = beam(None, max(1, min(log_int(rng, 1, 16), 64 // beams, 8192000 // (beams * vocab), 32000 * 8 * 128 // (held * kv * dim * beams))), beams, vocab, held, kv, dim,
                 rng.choice(["f16", "bf16", "f32"]))
    c.pop("name", None)
    return c


def lengths_of(c, held):
    """Rows that each sequence holds: `held` in the first, down to about half of it in the last."""
    n = c.get("seqs") or c["groups"] * c["beams"]
    if c["kind"] == "beam":
        return [max(1, held - (s // c["beams"]) * held // (2 * c["groups"])) for s in range(n)]
    return [held - s * held // (2 * n) for s in range(n)]


# ------------------------------------------------------------------ inputs
class Values:
    """Random tensors on the GPU, made from the seed and their order alone."""

    def __init__(self, seed):
        self.seed, self.made = seed, 0

    def generator(self):
        self.made += 1
        return torch.Generator(device="cuda").manual_seed(self.seed * 100003 + self.made)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=self.generator(), device="cuda").mul_(std).to(dtype)


def whole(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def seven_bits(s):
    """Non-negative binary32 values rounded to 7 significant bits, ties to even."""
    bits = s.view(torch.int32)
    return ((bits + 0xFFFF + ((bits >> 17) & 1)) & ~0x1FFFF).view(torch.float32)


def to_four_bits(x, block):
    """Codes 0 .. 15 (as binary32) and half scales of binary32 rows."""
    b = x.unflatten(-1, (-1, block))
    scale = seven_bits(b.abs().amax(-1) / torch.full((), 7.5, device=x.device)).clamp(max=8704.0).half()
    s = scale.float().unsqueeze(-1)
    code = torch.where(s > 0, torch.floor(b / s + 8.0).clamp(0.0, 15.0), torch.full((), 8.0, device=x.device))
    return code.flatten(-2), scale


def packed(code):
    """The row's bytes of codes."""
    words = code.to(torch.uint8).unflatten(-1, (-1, 4, 8)).transpose(-3, -2).flatten(-3)
    return (words[..., 0::2] | (words[..., 1::2] << 4)).contiguous()


def unpacked(codes):
    """Codes 0 .. 15 of a row's bytes, in the order of the dimensions."""
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return nibbles.unflatten(-1, (4, -1, 8)).transpose(-3, -2).flatten(-3)


def prepare(c, seed):
    v, kind = Values(seed), c["kind"]
    s = {"case": c}
    if kind in ("append", "attend"):
        t, seqs, rows, kv, dim, block = TYPES[c["dtype"]], c["seqs"], c["rows"], c["kv"], c["dim"], c["block"]
        context = c["held"] + rows + 5
        s["context"], s["lengths"] = context, whole(lengths_of(c, c["held"]))
        s["q"] = v.normal(seqs * rows, c["heads"] * dim, dtype=t)
        s["scales"] = [torch.zeros(seqs, kv, context, dim // block, dtype=torch.float16, device="cuda") for _ in range(2)]
        s["codes"] = [torch.zeros(seqs, kv, context, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    if kind == "append":
        # keys have channels that are several times larger than the others
        big = 1.0 + 4.0 * (torch.rand(kv * dim, generator=v.generator(), device="cuda") < 0.03)
        s["k"] = (v.normal(seqs * rows, kv * dim) * big).to(t)
        s["v"] = v.normal(seqs * rows, kv * dim, std=0.5, dtype=t)
        s["positions"] = s["lengths"] + c["shift"]
        s["q_out"] = torch.empty_like(s["q"])
        s["back"] = [torch.empty(seqs, kv, rows, dim, dtype=t, device="cuda") for _ in range(2)]
    elif kind == "attend":
        for one in range(seqs):
            for which in range(2):
                code, scale = to_four_bits(v.normal(kv, context, dim), block)
                s["codes"][which][one], s["scales"][which][one] = packed(code), scale
        s["out"] = torch.empty_like(s["q"])
        s["weights"] = torch.zeros(seqs, kv, context, device="cuda") if c["weights"] else None
    elif kind == "evict":
        seqs, kv, held, keep, dim = c["seqs"], c["kv"], c["held"], c["keep"], c["dim"]
        s["lengths"] = whole(lengths_of(c, held))
        s["planes"] = [v.normal(seqs, kv, held, dim, dtype=torch.float16) for _ in range(2)]
        s["weights"] = torch.exp(2.0 * v.normal(seqs, kv, held))  # a few rows receive most of the weight
        s["planes"].append(s["weights"].unsqueeze(-1))
        s["kept"] = torch.zeros(seqs, kv, keep, dtype=torch.int32, device="cuda")
        s["left"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        s["to"] = [torch.zeros(seqs, kv, keep, p.shape[-1], dtype=p.dtype, device="cuda") for p in s["planes"]]
    else:
        groups, beams, kv, held, dim = c["groups"], c["beams"], c["kv"], c["held"], c["dim"]
        n = groups * beams
        s["logits"] = v.normal(n, c["vocab"], std=2.5, dtype=TYPES[c["dtype"]])
        s["scores"] = v.normal(groups, beams, std=1.0) - 20.0
        s["lengths"] = whole(lengths_of(c, held))
        s["planes"] = [v.normal(n, kv, held, dim, dtype=torch.float16) for _ in range(2)]
        s["to"] = [torch.zeros_like(p) for p in s["planes"]]
        s["parents"], s["tokens"] = (torch.zeros(groups, beams, dtype=torch.int32, device="cuda") for _ in range(2))
        s["new_scores"] = torch.zeros(groups, beams, device="cuda")
    return s


# ------------------------------------------------------------------ the plain forms
def angles(positions, rows, dim, theta):
    """Rotation angles of `rows` positions behind each start, in 64 bits: [sequences * rows, dim / 2]."""
    at = (positions.double().unsqueeze(1) + torch.arange(rows, dtype=torch.float64, device="cuda")).reshape(-1, 1)
    return at * torch.pow(theta, -torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)


def rotated(x, dim, cos, sin):
    """Neighbouring pairs of every head, rotated in binary32."""
    p = x.float().unflatten(-1, (-1, dim // 2, 2))
    a, b, c, s = p[..., 0], p[..., 1], cos.unsqueeze(1), sin.unsqueeze(1)
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def plain_append(s):
    c = s["case"]
    seqs, rows, kv, dim = c["seqs"], c["rows"], c["kv"], c["dim"]
    a = angles(s["positions"], rows, dim, c["theta"])
    cos, sin = a.cos().float(), a.sin().float()
    s["q_out"].copy_(rotated(s["q"], dim, cos, sin).flatten(1))
    at = (s["lengths"].long().unsqueeze(1) + torch.arange(rows, device="cuda")).view(seqs, 1, rows, 1)
    new = (rotated(s["k"], dim, cos, sin), s["v"].float().unflatten(-1, (kv, dim)))
    for which in range(2):
        code, scale = to_four_bits(new[which].view(seqs, rows, kv, dim).transpose(1, 2), c["block"])
        s["codes"][which].scatter_(2, at.expand(-1, kv, -1, dim // 2), packed(code))
        s["scales"][which].scatter_(2, at.expand(-1, kv, -1, dim // c["block"]), scale)
        held = unpacked(s["codes"][which].gather(2, at.expand(-1, kv, -1, dim // 2))).float() - 7.5
        scales = s["scales"][which].gather(2, at.expand(-1, kv, -1, dim // c["block"])).float()
        s["back"][which].copy_((held.unflatten(-1, (-1, c["block"])) * scales.unsqueeze(-1)).flatten(-2))
    return {"q": s["q_out"], "k": s["back"][0], "v": s["back"][1]}


def plain_values(s, which):
    """Keys or values as the codes stand for them, in binary32: [sequences, kv, context, dim]."""
    held = unpacked(s["codes"][which]).float() - 7.5
    return (held.unflatten(-1, (-1, s["case"]["block"])) * s["scales"][which].float().unsqueeze(-1)).flatten(-2)


def plain_attend(s):
    c = s["case"]
    seqs, rows, kv, dim, context = c["seqs"], c["rows"], c["kv"], c["dim"], s["context"]
    group = c["heads"] // kv
    q = s["q"].float().view(seqs, rows, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * rows, dim)
    scores = torch.matmul(q, plain_values(s, 0).transpose(2, 3)).view(seqs, kv, group, rows, context) / math.sqrt(dim)
    seen = torch.arange(context, device="cuda") <= s["lengths"].view(-1, 1, 1) + torch.arange(rows, device="cuda").view(1, -1, 1)
    scores = torch.where(seen.view(seqs, 1, 1, rows, context), scores, torch.full((), -math.inf, device="cuda"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, kv, group * rows, context), plain_values(s, 1)).view(seqs, kv, group, rows, dim)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(seqs * rows, -1))
    if c["weights"]:
        s["weights"].copy_(p.double().sum((2, 3)))
    return {"out": s["out"], "weights": s["weights"]} if c["weights"] else {"out": s["out"]}


def plain_evict(s):
    c = s["case"]
    keep, recent = c["keep"], c["recent"]
    at, held = torch.arange(c["held"], device="cuda"), s["lengths"].view(-1, 1, 1)
    w = torch.where(at < held, s["weights"], torch.full((), -1.0, device="cuda"))
    w = torch.where((at >= held - recent) & (at < held), torch.full((), math.inf, device="cuda"), w)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    rows = torch.sort(torch.where(best < held, best, torch.full((), c["held"], dtype=best.dtype, device="cuda")), dim=-1).values
    there = rows < held
    s["kept"].copy_(torch.where(there, rows, torch.full((), -1, dtype=rows.dtype, device="cuda")))
    s["left"].copy_(s["lengths"].clamp(max=keep))
    for p, to in zip(s["planes"], s["to"]):
        moved = p.gather(2, rows.clamp(max=c["held"] - 1).unsqueeze(-1).expand(-1, -1, -1, p.shape[-1]))
        to.copy_(torch.where(there.unsqueeze(-1), moved, to))
    return {"kept": s["kept"], "left": s["left"], "keys": s["to"][0], "values": s["to"][1], "weights": s["to"][2]}


def plain_beam(s):
    c = s["case"]
    groups, beams, vocab = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    score = x - (torch.log(torch.exp(x - top).sum(-1, keepdim=True)) + top)
    score = (score.view(groups, beams, vocab) + s["scores"].double().unsqueeze(-1)).flatten(1)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    s["parents"].copy_(at[:, :beams] // vocab)
    s["tokens"].copy_(at[:, :beams] % vocab)
    s["new_scores"].copy_(best[:, :beams])
    parent = (s["parents"].long() + beams * torch.arange(groups, device="cuda").unsqueeze(1)).flatten()
    there = (torch.arange(c["held"], device="cuda") < s["lengths"][parent].unsqueeze(-1)).view(-1, 1, c["held"], 1)
    for p, to in zip(s["planes"], s["to"]):
        to.copy_(torch.where(there, p.index_select(0, parent), to))
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["new_scores"], "keys": s["to"][0], "values": s["to"][1]}


# ------------------------------------------------------------------ the library's operators
def pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def row_bytes(tensors):
    return (ctypes.c_int * len(tensors))(*[t.shape[-1] * t.element_size() for t in tensors])


def own_append(s, lib, check, stream):
    c = s["case"]
    seqs, rows, kv, dim, block, t = c["seqs"], c["rows"], c["kv"], c["dim"], c["block"], NUMBER[c["dtype"]]
    planes = [p.data_ptr() for pair in zip(s["codes"], s["scales"]) for p in pair]
    check(lib.lcu_cache4_append(*planes, s["q_out"].data_ptr(), s["q"].data_ptr(), c["heads"] * dim, s["k"].data_ptr(), s["v"].data_ptr(), kv * dim,
                                s["lengths"].data_ptr(), s["positions"].data_ptr(), seqs, rows, c["heads"], kv, dim, block, s["context"], c["theta"], t, stream))
    check(lib.lcu_cache4_read(s["back"][0].data_ptr(), s["back"][1].data_ptr(), *planes, s["lengths"].data_ptr(), seqs, rows, kv, dim, block, s["context"], t, stream))
    return {"q": s["q_out"], "k": s["back"][0], "v": s["back"][1]}


def own_attend(s, lib, check, stream):
    c = s["case"]
    seqs, rows, heads, kv, dim, context = c["seqs"], c["rows"], c["heads"], c["kv"], c["dim"], s["context"]
    if "workspace" not in s:
        need = lib.lcu_attention_cache4_workspace(seqs, rows, heads, kv, dim, c["held"] + rows, int(c["weights"]))
        s["workspace"] = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    weights = s["weights"].data_ptr() if c["weights"] else None
    planes = [p.data_ptr() for pair in zip(s["codes"], s["scales"]) for p in pair]
    check(lib.lcu_attention_cache4(s["out"].data_ptr(), heads * dim, weights, 0.0, s["q"].data_ptr(), heads * dim, *planes, s["lengths"].data_ptr(), seqs, rows,
                                   heads, kv, dim, c["block"], context, c["held"] + rows, NUMBER[c["dtype"]], s["workspace"].data_ptr(), s["workspace"].numel(),
                                   stream))
    return {"out": s["out"], "weights": s["weights"]} if c["weights"] else {"out": s["out"]}


def own_evict(s, lib, check, stream):
    c = s["case"]
    check(lib.lcu_cache_evict(pointers(s["to"]), pointers(s["planes"]), row_bytes(s["to"]), len(s["to"]), s["weights"].data_ptr(), s["kept"].data_ptr(),
                              s["left"].data_ptr(), s["lengths"].data_ptr(), c["seqs"], c["kv"], c["held"], c["keep"], c["keep"], c["recent"], stream))
    return {"kept": s["kept"], "left": s["left"], "keys": s["to"][0], "values": s["to"][1], "weights": s["to"][2]}


def own_beam(s, lib, check, stream):
    c = s["case"]
    groups, beams, vocab = c["groups"], c["beams"], c["vocab"]
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(16, lib.lcu_beam_select_workspace(groups, beams, vocab, beams)), dtype=torch.uint8, device="cuda")
    check(lib.lcu_beam_select(s["parents"].data_ptr(), s["tokens"].data_ptr(), s["new_scores"].data_ptr(), s["logits"].data_ptr(), vocab, NUMBER[c["dtype"]],
                              s["scores"].data_ptr(), groups, beams, vocab, beams, s["workspace"].data_ptr(), s["workspace"].numel(), stream))
    check(lib.lcu_cache_reorder(pointers(s["to"]), pointers(s["planes"]), row_bytes(s["to"]), len(s["to"]), s["parents"].data_ptr(), s["lengths"].data_ptr(), groups,
                                beams, c["kv"], c["held"], stream))
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["new_scores"], "keys": s["to"][0], "values": s["to"][1]}


PLAIN = {"append": plain_append, "attend": plain_attend, "evict": plain_evict, "beam": plain_beam}
OWN = {"append": own_append, "attend": own_attend, "evict": own_evict, "beam": own_beam}


def run(s):
    if own:
        lcu = library()
        return OWN[s["case"]["kind"]](s, lcu.lib, lcu.check, torch.cuda.current_stream().cuda_stream)
    return PLAIN[s["case"]["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    kind, dim = c["kind"], c["dim"]
    if kind in ("append", "attend"):
        row = c["kv"] * (dim // 2 + 2 * dim // c["block"])  # codes and scales of the keys, or the values, of one position
        tokens, lengths = c["seqs"] * c["rows"], lengths_of(c, c["held"])
    if kind == "append":
        # queries in and out, keys and values in, written to the cache, read back
        return {"bytes": tokens * (2 * 2 * c["heads"] * dim + 2 * 2 * c["kv"] * dim + 2 * 2 * row + 2 * 2 * c["kv"] * dim),
                "flops": tokens * dim * (3 * (c["heads"] + c["kv"]) + 6 * c["kv"])}
    if kind == "attend":
        seen = sum(n + c["rows"] for n in lengths)
        pairs = sum(c["rows"] * n + c["rows"] * (c["rows"] + 1) // 2 for n in lengths) * c["heads"]
        weights = 4 * seen * c["kv"] if c["weights"] else 0
        return {"bytes": 2 * 2 * tokens * c["heads"] * dim + 2 * seen * row + weights, "flops": 4 * pairs * dim}
    if kind == "evict":
        lengths = lengths_of(c, c["held"])
        moved = sum(min(n, c["keep"]) for n in lengths)
        return {"bytes": c["kv"] * (4 * sum(lengths) + 2 * moved * (2 * 2 * dim + 4) + 4 * c["seqs"] * c["keep"]), "flops": 0}
    n = c["groups"] * c["beams"]
    size = {"f16": 2, "bf16": 2, "f32": 4}[c["dtype"]]
    # (which beams are read is in the data: each new beam's rows are read and written once)
    return {"bytes": n * c["vocab"] * size + 16 * n + 2 * sum(lengths_of(c, c["held"])) * c["kv"] * 2 * 2 * dim, "flops": 4 * n * c["vocab"]}


# ------------------------------------------------------------------ the outputs in 64 bits
def exact_four_bits(x, block):
    """Values that the rows of x [..., dim] (binary64) are held as."""
    out = np.empty_like(x)
    for b in range(0, x.shape[-1], block):
        part = x[..., b:b + block]
        mantissa, exponent = np.frexp(np.abs(part).max(-1) / 7.5)
        scale = np.minimum(np.ldexp(np.rint(mantissa * 128.0) / 128.0, exponent), 8704.0).astype(np.float16).astype(np.float64)[..., None]
        safe = np.where(scale > 0, scale, 1.0)
        out[..., b:b + block] = (np.clip(np.floor(part / safe) + 8.0, 0.0, 15.0) - 7.5) * scale
    return out


def exact_append(s):
    c = s["case"]
    seqs, rows, dim = c["seqs"], c["rows"], c["dim"]
    at = (s["positions"].cpu().numpy().astype(np.float64)[:, None] + np.arange(rows)).reshape(-1, 1, 1)
    turn = np.exp(1j * at * c["theta"] ** (-np.arange(0, dim, 2) / dim))

    def turned(x, heads):
        z = x.double().cpu().numpy().reshape(-1, heads, dim // 2, 2)
        z = (z[..., 0] + 1j * z[..., 1]) * turn
        return np.stack((z.real, z.imag), -1).reshape(-1, heads, dim)

    def held(x):
        return torch.from_numpy(exact_four_bits(x.reshape(seqs, rows, c["kv"], dim).transpose(0, 2, 1, 3), c["block"]))

    return {"q": torch.from_numpy(turned(s["q"], c["heads"]).reshape(seqs * rows, -1)), "k": held(turned(s["k"], c["kv"])),
            "v": held(s["v"].double().cpu().numpy().reshape(-1, c["kv"], dim))}


def exact_attend(s):
    """Row by row of the definition: softmax over the visible keys, by log-sum-exp; head by head, so that the scores fit."""
    c = s["case"]
    seqs, rows, kv, dim, block = c["seqs"], c["rows"], c["kv"], c["dim"], c["block"]
    group, groups = c["heads"] // kv, dim // 32
    word_of = [(d % 32) // 8 * groups + d // 32 for d in range(dim)]
    byte = torch.tensor([w * 4 + d % 8 // 2 for d, w in enumerate(word_of)], device="cuda")
    odd = torch.tensor([d % 2 for d in range(dim)], device="cuda")
    out = torch.zeros(seqs, rows, kv, group, dim, dtype=torch.float64, device="cuda")
    weights = torch.zeros(seqs, kv, s["context"], dtype=torch.float64, device="cuda")
    for one, n in enumerate(s["lengths"].tolist()):
        for h in range(kv):
            kept = []
            for which in range(2):
                raw = s["codes"][which][one, h, :n + rows].index_select(1, byte).int()
                code = torch.where(odd == 1, raw >> 4, raw & 15).double()
                kept.append((2 * code - 15) * s["scales"][which][one, h, :n + rows].double().repeat_interleave(block, -1) / 2)
            hidden = torch.ones(rows, n + rows, dtype=torch.bool, device="cuda").triu(n + 1)
            for g in range(group):
                q = s["q"][one * rows:(one + 1) * rows].view(rows, kv, group, dim)[:, h, g].double()
                a = (q @ kept[0].T * dim ** -0.5).masked_fill(hidden, -math.inf)
                p = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
                out[one, :, h, g] = p @ kept[1]
                weights[one, h, :n + rows] += p.sum(0)
    out = out.view(seqs * rows, -1)
    return {"out": out, "weights": weights} if c["weights"] else {"out": out}


def exact_beam(s):
    """Log-probabilities by log-sum-exp, the best one after another."""
    c = s["case"]
    total = torch.log_softmax(s["logits"].double(), -1).view(c["groups"], -1) + s["scores"].double().repeat_interleave(c["vocab"], 1)
    scores = []
    for _ in range(c["beams"]):
        best, at = total.max(-1)
        scores.append(best)
        total.scatter_(1, at.unsqueeze(1), -math.inf)
    return {"parents": None, "tokens": None, "scores": torch.stack(scores, 1), "keys": None, "values": None}


def exact(c, seed):
    if c["kind"] == "evict":
        return None  # (rows are moved, nothing is computed)
    s = prepare(c, seed)
    return {"append": exact_append, "attend": exact_attend, "beam": exact_beam}[c["kind"]](s)
