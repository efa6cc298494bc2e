"""The attention operators as cases that can be timed and compared: the paged key-value cache's write and read, the
attention of new tokens over it, and the attention over packed prompts.

Shapes are those of the repository's trunk: q 4096 with k, v 512 (32 / 4 heads of 128, 16 / 2 of 256, 64 / 8 of 64) and
q 10240 with k, v 640 (80 / 5 heads of 128); activations f32 as the linears write them, or 16 bits.

A case's sequence lengths follow from the case alone (`_lens`): log-uniform from lo to hi, so that batches are ragged.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64  # tokens of a cache page
TYPES = {"F32": torch.float32, "BF16": torch.bfloat16, "F16": torch.float16}
HEADS = [(32, 4, 128), (16, 2, 256), (64, 8, 64), (80, 5, 128), (8, 8, 128), (20, 4, 64), (24, 2, 256)]


def listed():
    return [
        # one decode step's new tokens of 64 sequences into an 8-bit cache
        {"name": "write_step_i8", "kind": "write", "n": 64, "lo": 1, "hi": 4000, "tlo": 1, "thi": 1, "heads": 4,
         "dim": 128, "cache": "I8", "type": "F32", "mix": 1},
        # the prefill chunk of a batch of prompts into a 16-bit cache
        {"name": "write_prompt_bf16", "kind": "write", "n": 5, "lo": 300, "hi": 2000, "tlo": 300, "thi": 2000, "heads": 4,
         "dim": 128, "cache": "BF16", "type": "F32", "mix": 2},
        # the tokens of a short conversation brought back, and the history of three long ones in front of their next chunk
        {"name": "read_short_f16", "kind": "read", "n": 1, "lo": 100, "hi": 100, "heads": 2, "dim": 256, "cache": "F16",
         "type": "F32", "mix": 3},
        {"name": "read_history_i8", "kind": "read", "n": 3, "lo": 5000, "hi": 20000, "heads": 4, "dim": 128,
         "cache": "I8", "type": "BF16", "mix": 4},
        # the first words of an answer: one sequence, little in the cache, latency counts
        {"name": "decode_1seq_short", "kind": "decode", "n": 1, "lo": 37, "hi": 37, "tlo": 1, "thi": 1, "qheads": 32,
         "heads": 4, "dim": 128, "cache": "BF16", "type": "F32", "mix": 5},
        # a serving batch in mid-conversation, 8-bit cache
        {"name": "decode_batch_i8", "kind": "decode", "n": 48, "lo": 200, "hi": 4000, "tlo": 1, "thi": 1, "qheads": 32,
         "heads": 4, "dim": 128, "cache": "I8", "type": "F32", "mix": 6},
        # one long document, two key heads: the cache's length is all there is to split
        {"name": "decode_long_bf16", "kind": "decode", "n": 1, "lo": 131072, "hi": 131072, "tlo": 1, "thi": 1,
         "qheads": 16, "heads": 2, "dim": 256, "cache": "BF16", "type": "BF16", "mix": 7},
        # drafts of 16 sequences verified together, between one and six each, sixteen query heads to a key head
        {"name": "decode_drafts_bf16", "kind": "decode", "n": 16, "lo": 1000, "hi": 16000, "tlo": 1, "thi": 6,
         "qheads": 80, "heads": 5, "dim": 128, "cache": "BF16", "type": "F32", "mix": 8},
        # a one-line prompt
        {"name": "prompt_short_f32", "kind": "prompt", "n": 1, "lo": 33, "hi": 33, "back": 0, "qheads": 32, "heads": 4,
         "dim": 128, "type": "F32", "mix": 9},
        # prompts of several users packed into one call
        {"name": "prompt_packed_bf16", "kind": "prompt", "n": 9, "lo": 40, "hi": 1500, "back": 0, "qheads": 32, "heads": 4,
         "dim": 128, "type": "BF16", "mix": 10},
        # a later chunk of a long document: its 2048 tokens see 14000 earlier ones as well
        {"name": "prompt_chunk_f16", "kind": "prompt", "n": 1, "lo": 2048, "hi": 2048, "back": 14000, "qheads": 16,
         "heads": 2, "dim": 256, "type": "F16", "mix": 11},
        # a full chunk of 4096 in the trunk's own 32-bit activations
        {"name": "prompt_4096_f32", "kind": "prompt", "n": 1, "lo": 4096, "hi": 4096, "back": 0, "qheads": 64, "heads": 8,
         "dim": 64, "type": "F32", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    qh, h, d = rng.choice(HEADS)
    c = {"kind": kind, "heads": h, "dim": d, "mix": rng.randrange(1 << 20), "type": rng.choice(["F32", "BF16", "F16"])}
    if kind in ("write", "read", "decode"):
        c["cache"] = rng.choice(["BF16", "F16", "I8"])
    if kind == "write":
        n = _log_int(rng, 1, 200)
        hi = _log_int(rng, 1, 8000 // n)
        c.update({"n": n, "hi": hi + _log_int(rng, 1, 2000), "lo": max(1, hi // 8), "tlo": max(1, hi // 8), "thi": hi})
    elif kind == "read":
        n = _log_int(rng, 1, 100)
        hi = _log_int(rng, 8, 40000 // n)
        c.update({"n": n, "hi": hi, "lo": max(1, hi // 8)})
    elif kind == "decode":
        n = _log_int(rng, 1, 200)
        hi = _log_int(rng, 4, max(200, 130000 * 256 // (n * h * d)))
        c.update({"n": n, "hi": hi, "lo": max(1, hi // 10), "tlo": 1, "thi": rng.choice([1, 1, 1, 4, 8]), "qheads": qh})
    else:
        n = _log_int(rng, 1, 24)
        hi = _log_int(rng, 4, 4000 // n)
        c.update({"n": n, "hi": hi, "lo": max(1, hi // 8), "back": rng.choice([0, 0, _log_int(rng, 1, 4000)]) if n <= 2 else 0,
                  "qheads": qh})
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def _lens(case):
    """tokens of each sequence in the cache (or in the prompt), and how many of them are this call's rows"""
    r = random.Random(case["mix"])
    lens = [_log_int(r, case["lo"], case["hi"]) for _ in range(case["n"])]
    if case["kind"] == "read":
        return lens, lens
    if case["kind"] == "prompt":
        return [v + case["back"] for v in lens], lens
    return lens, [min(v, r.randint(case["tlo"], case["thi"])) if case["kind"] == "decode" else
                  min(v, _log_int(r, case["tlo"], case["thi"])) for v in lens]


def _inputs(case, seed):
    """k, v (and q) rows as the trunk's linears hand them on; a key's channels differ in size. For the cases on a cache,
    also its page table: a pool's pages in the order in which they happened to be free."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    lens, new = _lens(case)
    H, D, n = case["heads"], case["dim"], case["n"]
    d = {"lens": lens, "new": new}
    t = TYPES[case["type"]]
    total = sum(new) if case["kind"] == "write" else sum(lens)
    d["k"] = normal(total, H, D) * torch.exp(0.4 * normal(1, H, D))
    d["v"] = normal(total, H, D)
    if case["kind"] in ("write", "prompt"):
        d["k"], d["v"] = d["k"].to(t), d["v"].to(t)
    if case["kind"] in ("decode", "prompt"):
        d["q"] = normal(sum(new), case["qheads"], D).to(t)
    if case["kind"] != "prompt":
        per = [-(-v // PAGE) for v in lens]
        d["pages"], d["ldt"] = sum(per) + 8, max(per)
        ids = torch.randperm(d["pages"], generator=g, device="cuda").int()
        table = torch.zeros(n, d["ldt"], dtype=torch.int32, device="cuda")
        at = 0
        for b, p in enumerate(per):
            table[b, :p] = ids[at:at + p]
            at += p
        d["table"] = table
    d["lens_t"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    d["rows_t"] = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device="cuda")
    d["krows_t"] = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
    return d


# ---------------------------------------------------------------------------------------------------- a program's side
_engine = None


def _eng():
    global _engine
    if _engine is None:
        import ijah_amd
        _engine = ijah_amd.load_engine()
    return _engine


class _Bytes:
    """A device buffer's memory, for torch (as bytes: it has no code for bf16)."""

    def __init__(self, buf, nbytes):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "version": 3, "strides": None,
                                         "data": (int(buf.gpu_address()), False)}


def _like(*shape, dtype):
    """A device buffer of the library and torch's view of it."""
    n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    b = _eng().alloc(n)
    return b, torch.as_tensor(_Bytes(b, n), device="cuda").view(dtype).reshape(shape)


def _buf(t):
    b, v = _like(*t.shape, dtype=t.dtype)
    v.copy_(t)
    return b


def prepare(case, seed):
    """A program of this library holds its activations, tables and cache in the library's buffers, so that is what `own`
    makes of the same inputs here."""
    d, kind = _inputs(case, seed), case["kind"]
    H, D, t, R = case["heads"], case["dim"], TYPES[case["type"]], sum(d["new"])
    s = {"case": case, "R": R, "scale": 1 / math.sqrt(D), "maxlen": max(d["lens"]), "maxnew": max(d["new"])}
    if own:
        from ijah_amd.engine import KvSeqs
        rows, lens = _buf(d["rows_t"]), _buf(d["lens_t"])
        if kind == "prompt":
            s["q"], s["k"], s["v"] = _buf(d["q"]), _buf(d["k"]), _buf(d["v"])
            s["rows"], s["krows"], s["Rk"] = rows, _buf(d["krows_t"]), sum(d["lens"])
        else:
            table = _buf(d["table"])
            s["seqs"] = KvSeqs(case["n"], d["ldt"], table, lens, rows)
            s["cache"] = _eng().kv_create(1, d["pages"], H, D, case["cache"])
            if kind == "write":
                s["k"], s["v"] = _buf(d["k"]), _buf(d["v"])
            else:  # what earlier steps have written
                whole = KvSeqs(case["n"], d["ldt"], table, lens, _buf(d["krows_t"]))
                k, v = _buf(d["k"]), _buf(d["v"])
                torch.cuda.synchronize()
                s["cache"].write_bufs(0, whole, sum(d["lens"]), k, v)
                _eng().sync()  # the rows' buffers go with this call
            if kind == "decode":
                s["q"] = _buf(d["q"])
        if kind in ("write", "read"):
            s["ko"], kv = _like(R, H, D, dtype=t)
            s["vo"], vv = _like(R, H, D, dtype=t)
            s["views"] = [kv, vv]
        else:
            s["o"], ov = _like(R, case["qheads"], D, dtype=t)
            s["views"] = [ov]
    else:
        s.update({k: d[k] for k in ("lens_t", "rows_t", "krows_t", "table", "q") if k in d})
        if kind in ("write", "prompt"):
            s["k"], s["v"] = d["k"], d["v"]
        if kind != "prompt":
            held = {"I8": torch.int8, **TYPES}[case["cache"]]
            s["cache"] = {x: torch.zeros(d["pages"] * PAGE, H, D, dtype=held, device="cuda") for x in "kv"}
            s["cache"].update({x + "s": torch.zeros(d["pages"] * PAGE, H, device="cuda") for x in "kv"})
            if kind != "write":
                at = _places(d["table"], d["lens_t"], d["krows_t"], sum(d["lens"]))
                _store(s["cache"], "k", at, d["k"])
                _store(s["cache"], "v", at, d["v"])
    torch.cuda.synchronize()
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case, kind, R = s["case"], s["case"]["kind"], s["R"]
    if kind == "write":  # the values written, read back: the cache's own layout is its own affair
        s["cache"].write_bufs(0, s["seqs"], R, s["k"], s["v"], dtype=case["type"])
        s["cache"].read_bufs(0, s["seqs"], R, s["ko"], s["vo"], dtype=case["type"])
    elif kind == "read":
        s["cache"].read_bufs(0, s["seqs"], R, s["ko"], s["vo"], dtype=case["type"])
    elif kind == "decode":
        s["cache"].attend_bufs(0, s["seqs"], R, case["qheads"], s["q"], s["o"], dtype=case["type"], scale=s["scale"])
    else:
        _eng().attn_prompt_bufs(case["n"], s["rows"], s["krows"], R, s["Rk"], case["qheads"], case["heads"], case["dim"],
                                s["q"], s["k"], s["v"], s["o"], dtype=case["type"], scale=s["scale"])
    return s["views"]


# ---------------------------------------------------------------------------------------------------- the plain forms
def _of_rows(rows_t, R):
    """each row's sequence, and its number among the sequence's rows"""
    r = torch.arange(R, device="cuda")
    b = torch.searchsorted(rows_t, r.int(), right=True) - 1
    return b, r - rows_t[b]


def _places(table, lens_t, rows_t, R):
    """each row's token in the cache: the sequence's newest rows, the last one at its length - 1"""
    b, i = _of_rows(rows_t, R)
    p = lens_t[b] - (rows_t[b + 1] - rows_t[b]) + i
    return table[b, p // PAGE].long() * PAGE + p % PAGE


def _store(cache, x, at, rows):
    rows = rows.float()
    if cache[x].dtype == torch.int8:
        s = rows.abs().amax(-1) / 127
        cache[x + "s"][at] = s
        rows = torch.round(rows / torch.where(s > 0, s, 1.0)[..., None]).clamp(-127, 127)
    cache[x][at] = rows.to(cache[x].dtype)


def _load(cache, x, at):
    c = cache[x][at].float()
    return c * cache[x + "s"][at][..., None] if cache[x].dtype == torch.int8 else c


def _attend(q, k, v, mask, scale):
    """q f32 [..., H, rows, D], k, v f32 [..., H, keys, D], mask [..., 1, rows, keys]; a row that sees no key is zero"""
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~mask, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(l == 0, 1.0, l)


def _run_plain(s):
    case, kind, R = s["case"], s["case"]["kind"], s["R"]
    t, H, D = TYPES[case["type"]], case["heads"], case["dim"]
    if kind in ("write", "read"):
        at = _places(s["table"], s["lens_t"], s["rows_t"], R)
        if kind == "write":
            _store(s["cache"], "k", at, s["k"])
            _store(s["cache"], "v", at, s["v"])
        return [_load(s["cache"], x, at).to(t) for x in "kv"]
    Hq = case["qheads"]
    g = Hq // H
    if kind == "decode":
        n, T, L = case["n"], s["maxnew"], s["maxlen"]
        b, i = _of_rows(s["rows_t"], R)
        q = torch.zeros(n, T, Hq, D, device="cuda")
        q[b, i] = s["q"].float()
        q = q.reshape(n, T, H, g, D).permute(0, 2, 3, 1, 4).reshape(n, H, g * T, D)
        j = torch.arange(L, device="cuda")
        at = s["table"][:, j // PAGE].long() * PAGE + j % PAGE
        k, v = (_load(s["cache"], x, at).permute(0, 2, 1, 3) for x in "kv")
        new = s["rows_t"][1:] - s["rows_t"][:-1]
        last = (s["lens_t"] - new)[:, None] + torch.arange(T, device="cuda")  # each row's own position
        mask = (j <= last[..., None]) & (j < s["lens_t"][:, None, None])
        mask = mask[:, None, None].expand(n, 1, g, T, L).reshape(n, 1, g * T, L)
        o = _attend(q, k, v, mask, s["scale"])
        return [o.reshape(n, H, g, T, D).permute(0, 3, 1, 2, 4).reshape(n, T, Hq, D)[b, i].to(t)]
    k, v = s["k"].float(), s["v"].float()
    bq, i = _of_rows(s["rows_t"], R)
    bk, j = _of_rows(s["krows_t"], k.shape[0])
    behind = ((s["krows_t"][1:] - s["krows_t"][:-1]) - (s["rows_t"][1:] - s["rows_t"][:-1]))[bq]
    mask = (bq[:, None] == bk) & (j <= (i + behind)[:, None])
    q = s["q"].float().reshape(R, H, g, D).permute(1, 2, 0, 3)
    o = _attend(q, k.permute(1, 0, 2)[:, None], v.permute(1, 0, 2)[:, None], mask, s["scale"])
    return [o.permute(2, 0, 1, 3).reshape(R, Hq, D).to(t)]


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    """what is read and written once; two operations for each product term of a visible pair"""
    lens, new = _lens(case)
    H, D, R = case["heads"], case["dim"], sum(new)
    e = 4 if case["type"] == "F32" else 2
    if case["kind"] == "prompt":
        Hq = case["qheads"]
        pairs = sum(m * (v - m) + m * (m + 1) / 2 for v, m in zip(lens, new))
        return {"bytes": float(e * D * (2 * R * Hq + 2 * sum(lens) * H)), "flops": float(4 * D * Hq * pairs)}
    c = 2 * H * (D + 4 if case["cache"] == "I8" else 2 * D)  # a token's keys and values in the cache
    if case["kind"] == "write":  # rows in, cache written, cache read, rows out
        return {"bytes": float(R * (2 * c + 4 * H * D * e)), "flops": float(6 * R * H * D)}
    if case["kind"] == "read":
        return {"bytes": float(R * (c + 2 * H * D * e)), "flops": float(2 * R * H * D)}
    Hq = case["qheads"]
    pairs = sum(m * (v - m) + m * (m + 1) / 2 for v, m in zip(lens, new))
    return {"bytes": float(sum(lens) * c + 2 * R * Hq * D * e), "flops": float(4 * D * Hq * pairs)}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _held(x, cache):
    """what the cache holds of f32 rows: the nearest 16-bit value, or the nearest of 255 steps of max / 127, where step and
    quotient are by definition 32-bit numbers (the 64-bit quotient would fall on the other side of a border now and then,
    and such a value is an input of what reads the cache)"""
    if cache != "I8":
        return x.to(TYPES[cache]).double()
    step = x.abs().amax(-1, keepdim=True) / 127
    q = torch.round(x / torch.where(step > 0, step, 1.0))
    return q.double() * step.double()


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    H, D = case["heads"], case["dim"]
    if kind in ("write", "read"):
        return [_held(d[x].float(), case["cache"]) for x in "kv"]
    k, v = d["k"], d["v"]
    if kind == "decode":
        k, v = _held(k, case["cache"]), _held(v, case["cache"])
    g = case["qheads"] // H
    out = torch.zeros(sum(d["new"]), case["qheads"], D, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for L, m in zip(d["lens"], d["new"]):  # a sequence, then a key head, then a piece of its rows at a time
        for h in range(H):
            kh, vh = k[k0:k0 + L, h].double(), v[k0:k0 + L, h].double()
            for r in range(0, m, 1024):
                c = min(1024, m - r)
                q = d["q"][q0 + r:q0 + r + c, h * g:(h + 1) * g].double().reshape(c * g, D)
                w = q @ kh.T / math.sqrt(D)
                seen = L - m + r + torch.arange(c, device="cuda").repeat_interleave(g)
                w = torch.where(torch.arange(L, device="cuda") <= seen[:, None], w, -math.inf)
                out[q0 + r:q0 + r + c, h * g:(h + 1) * g] = (torch.softmax(w, 1) @ vh).reshape(c, g, D)
        q0, k0 = q0 + m, k0 + L
    return [out]
