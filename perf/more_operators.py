"""Operators of long caches, as cases that can be timed and checked.

A cache that outgrows FP32 rows is held in 4 bits, or loses the rows that attention
hardly looks at:

  append   FP32 k and v rows into a cache of 4 bits (group 32), and the rows read back
  attn     attention over such a cache, with the weight that each key got if asked for
  weights  the weight that each key of an FP32 cache got
  evict    the rows to keep: the first, the latest, and the heaviest of the others

Sizes are a Gemma-4-E2B-shaped decoder's (8 query heads on one KV head, head dims 256
and 512, a 512-key window) or generic ones around them.
"""
import math

import numpy as np
import torch

own = False

HEADS, WINDOW, GROUP = 8, 512, 32


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # one token's k and v of a windowed layer, in the middle of a chat
        {"name": "append_token", "kind": "append", "n": 1, "hd": 256, "at": 1900},
        # a long prompt's rows of a layer that sees everything
        {"name": "append_prompt", "kind": "append", "n": 4000, "hd": 512, "at": 0},
        # one token in a windowed layer
        {"name": "attn_window", "kind": "attn", "rows": 1, "heads": HEADS, "hd": 256, "keys": 2778, "window": WINDOW, "weights": False},
        # one token after a document
        {"name": "attn_token", "kind": "attn", "rows": 1, "heads": HEADS, "hd": 512, "keys": 16001, "window": 0, "weights": False},
        # one token of a chat whose cache is thinned later: every key's weight is kept
        {"name": "attn_token_weights", "kind": "attn", "rows": 1, "heads": HEADS, "hd": 512, "keys": 32003, "window": 0, "weights": True},
        # one token at the end of a whole book
        {"name": "attn_far", "kind": "attn", "rows": 1, "heads": HEADS, "hd": 512, "keys": 131072, "window": 0, "weights": False},
        # a chunk of a prompt behind an earlier one
        {"name": "attn_prompt", "kind": "attn", "rows": 512, "heads": HEADS, "hd": 512, "keys": 4608, "window": 0, "weights": False},
        # a ragged chunk, with the keys' weights
        {"name": "attn_prompt_weights", "kind": "attn", "rows": 203, "heads": HEADS, "hd": 512, "keys": 2403, "window": 0, "weights": True},
        # one token over FP32 rows
        {"name": "weights_token", "kind": "weights", "rows": 1, "heads": HEADS, "hd": 512, "keys": 8001, "window": 0},
        # the last rows of a prompt, which say what of it will be looked at
        {"name": "weights_prompt", "kind": "weights", "rows": 256, "heads": HEADS, "hd": 512, "keys": 4096, "window": 0},
        # the three caches of the layers that see everything, 64 rows over their budget
        {"name": "evict_layers", "kind": "evict", "sets": 3, "len": 2112, "keep": 2048, "first": 4, "recent": 128},
        # a book's cache cut to a quarter
        {"name": "evict_book", "kind": "evict", "sets": 1, "len": 131072, "keep": 32768, "first": 4, "recent": 512},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "attn", "weights", "evict"])
    if kind == "append":
        return {"kind": kind, "n": _log(rng, 1, 4000), "hd": rng.choice([64, 128, 256, 256, 512, 512]), "at": rng.randint(0, 5000)}
    if kind == "evict":
        sets, n = rng.choice([1, 1, 2, 3, 7, 15]), _log(rng, 16, 131072)
        n = min(n, 131072 // sets)
        keep = rng.randint(max(2, n // 4), n)
        first = rng.randint(0, min(16, keep // 2))
        return {"kind": kind, "sets": sets, "len": n, "keep": keep, "first": first, "recent": rng.randint(0, min(512, keep - first))}
    rows = rng.choice([1, 1, _log(rng, 2, 512)]) if kind == "attn" else rng.choice([1, _log(rng, 2, 256)])
    most = (131072 if kind == "attn" else 16000) if rows <= 8 else (2048000 if kind == "attn" else 1000000) // rows
    keys = rows + _log(rng, 1, max(2, min(most, 131072) - rows))
    case = {"kind": kind, "rows": rows, "heads": rng.choice([1, 2, 3, 4, 6, 8, 8, 8]), "hd": rng.choice([64, 128, 256, 256, 512, 512]),
            "keys": keys, "window": rng.choice([0, 0, WINDOW, rng.randint(2, 1500)])}
    if kind == "attn":
        case["weights"] = rng.random() < 0.4
    return case


# ---- inputs ------------------------------------------------------------------

def _library():
    """The Python front end, initialised (its buffers and calls need the device)."""
    import os
    import sys
    if "g4hip" not in sys.modules:
        sys.path.insert(0, os.path.abspath("gemma4-js_amd"))
    import g4hip
    g4hip.init(0)
    return g4hip


class _Seen:
    """Memory of the library as torch sees it."""

    def __init__(self, ptr, shape, typestr):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr,
                                         "data": (ptr, False), "version": 2}


class _Held:
    """A tensor of the program: with the framework, in a buffer of its own memory."""

    def __init__(self, t):
        t = t.contiguous()
        self.t = t
        if own:
            g4 = _library()
            self.buf = g4.Buffer(t.numel() * t.element_size())
            g4.sync()  # a new buffer is filled with zeros on the library's queue
            code = {torch.float32: "<f4", torch.int32: "<i4", torch.bfloat16: "<i2"}[t.dtype]
            seen = torch.as_tensor(_Seen(self.buf.ptr, t.shape, code), device="cuda")
            self.t = seen.view(torch.bfloat16) if t.dtype == torch.bfloat16 else seen
            self.t.copy_(t)
            torch.cuda.synchronize()
            self.ptr = self.buf.ptr


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    return g


def _normal(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * sigma


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "evict":
        # sums of weights: a few rows that every token looks at, many that none does
        w = torch.exp(2.5 * _normal(g, case["sets"], case["len"]) - 3.0)
        return {"w": torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.05, torch.zeros_like(w), w)}
    hd = case["hd"]
    # normed rows: q.k of a few units, as trained q and k norms leave it
    at = 1.5 / math.sqrt(math.sqrt(hd))
    if kind == "append":
        return {"k": _normal(g, case["n"], hd, sigma=at), "v": _normal(g, case["n"], hd)}
    x = {"q": _normal(g, case["rows"], case["heads"], hd, sigma=at), "k": _normal(g, case["keys"], hd, sigma=at)}
    if kind == "attn":
        x["v"] = _normal(g, case["keys"], hd)
    if kind == "weights" or case["weights"]:
        # what earlier tokens left: of the size of what these add
        x["before"] = torch.exp(2.0 * _normal(g, case["keys"]) - 2.0) * (case["rows"] * case["heads"] / case["keys"])
    return x


def _blank(*shape, dtype=torch.float32):
    return _Held(torch.zeros(*shape, dtype=dtype, device="cuda"))


def _planes(rows, hd):
    """The four planes of a cache of 4 bits: codes and scales of k and v."""
    return {"k4": _blank(rows, hd // 8, dtype=torch.int32), "ks": _blank(rows, hd // GROUP, dtype=torch.bfloat16),
            "v4": _blank(rows, hd // 8, dtype=torch.int32), "vs": _blank(rows, hd // GROUP, dtype=torch.bfloat16)}


def prepare(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    st = {n: _Held(t) for n, t in x.items() if not (kind == "attn" and n in "kv")}
    st["case"] = case
    if kind == "append":
        st.update(_planes(case["at"] + case["n"], case["hd"]))
        st["k_back"], st["v_back"] = _blank(case["n"], case["hd"]), _blank(case["n"], case["hd"])
    elif kind == "attn":  # the cache, filled by earlier tokens
        for n, c, s in (("k", "k4", "ks"), ("v", "v4", "vs")):
            st[c], st[s] = (_Held(t) for t in _pack(x[n]))
        st["y"] = _blank(case["rows"], case["heads"], case["hd"])
    elif kind == "evict":
        st["rows"], st["kept"] = _blank(case["sets"], case["keep"], dtype=torch.int32), _blank(case["sets"], case["len"])
    if "before" in st:
        st["after"] = _blank(case["keys"])
    if own and "k4" in st:
        st["cache"] = _library().Kv4Cache(st["k4"].t.shape[0], case["hd"], [st[n] for n in ("k4", "ks", "v4", "vs")])
    return st


# ---- one pass ------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    kind = case["kind"]
    if kind == "append":
        n, at = case["n"], case["at"]
        st["k4"].t[at:at + n], st["ks"].t[at:at + n] = _pack(st["k"].t)
        st["v4"].t[at:at + n], st["vs"].t[at:at + n] = _pack(st["v"].t)
        return {"k": _unpack(st["k4"].t[at:at + n], st["ks"].t[at:at + n]),
                "v": _unpack(st["v4"].t[at:at + n], st["vs"].t[at:at + n])}
    if kind == "evict":
        return _heaviest(case, st["w"].t)
    # the keys that some row sees
    first = max(0, case["keys"] - case["rows"] - case["window"] + 1) if case["window"] else 0
    k = st["k"].t[first:] if kind == "weights" else _unpack(st["k4"].t[first:], st["ks"].t[first:])
    p, total = _weigh(case, st["q"].t, k, first)
    out = {}
    if kind == "attn":
        v = _unpack(st["v4"].t[first:], st["vs"].t[first:])
        out["y"] = ((p @ v) / total).view(case["rows"], case["heads"], case["hd"])
    if "before" in st:
        out["weights"] = st["before"].t.clone()
        out["weights"][first:] += (p / total).sum(0)
    return out


def _run_own(st):
    import g4hip
    case = st["case"]
    kind = case["kind"]
    if kind == "append":
        st["cache"].append(st["k"], st["v"], case["n"], case["at"])
        st["cache"].read(case["at"], case["n"], st["k_back"], st["v_back"])
        return {"k": st["k_back"].t, "v": st["v_back"].t}
    if kind == "evict":
        g4hip.cache_evict(st["w"], case["sets"], case["len"], case["keep"], case["first"], case["recent"],
                          st["rows"], st["kept"])
        return {"rows": st["rows"].t, "kept": st["kept"].t}
    rows, keys, window = case["rows"], case["keys"], case["window"]
    if kind == "weights":
        g4hip.attention_weights(st["q"], st["k"], rows, case["heads"], case["hd"], keys, keys - rows, window > 0,
                                window, st["after"], st["before"])
        return {"weights": st["after"].t}
    after = st.get("after")
    st["cache"].attention(st["q"], rows, case["heads"], keys, keys - rows, window > 0, window, st["y"], after,
                          st.get("before"))
    return {"y": st["y"].t, "weights": after.t} if after else {"y": st["y"].t}


def _pack(x):
    """Codes [n, hd / 8] and scales [n, hd / 32]: s = bf16(max |x| / 7), q = x / s to the nearest
    whole number within 7, stored as q + 8, eight to a word, the first one lowest."""
    g = x.view(x.shape[0], -1, GROUP)
    # (quotients in 64 bits: a value may lie next to the border of two codes)
    s = (g.abs().amax(2).double() / 7.0).float().bfloat16()
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = torch.round(g.double() / s.double()[:, :, None]).clamp(-7, 7).to(torch.int32) + 8
    shift = 4 * torch.arange(8, dtype=torch.int32, device=x.device)
    return (q.view(x.shape[0], -1, 8) << shift).sum(2, dtype=torch.int32), s


def _unpack(codes, scales):
    shift = 4 * torch.arange(8, dtype=torch.int32, device=codes.device)
    q = ((codes[:, :, None] >> shift) & 15).float() - 8.0
    return (q.view(codes.shape[0], -1, GROUP) * scales.float()[:, :, None]).view(codes.shape[0], -1)


def _weigh(case, q, k, first):
    """e^(q.k - the row's largest) of the keys from `first` on that a row sees, and the rows' sums."""
    rows, heads, window = case["rows"], case["heads"], case["window"]
    s = q.reshape(rows * heads, -1) @ k.T
    pos = torch.arange(case["keys"] - rows, case["keys"], device=q.device).repeat_interleave(heads)[:, None]
    at = torch.arange(first, case["keys"], device=q.device)[None, :]
    sees = at <= pos
    if window:
        sees = sees & (at > pos - window)
    s = s.masked_fill(~sees, -math.inf)
    p = torch.exp(s - s.amax(1, keepdim=True))
    return p, p.sum(1, keepdim=True)


def _heaviest(case, w):
    """The rows that stay, in their order, and their weights with zeros behind."""
    n, keep, first, recent = (case[x] for x in ("len", "keep", "first", "recent"))
    between = torch.sort(w[:, first:n - recent], dim=1, descending=True, stable=True).indices
    between = between[:, :keep - first - recent] + first
    ends = torch.cat([torch.arange(first, device=w.device), torch.arange(n - recent, n, device=w.device)])
    rows = torch.cat([between, ends[None].expand(w.shape[0], -1)], 1).sort(1).values
    kept = torch.zeros_like(w)
    kept[:, :keep] = w.gather(1, rows)
    return {"rows": rows.to(torch.int32), "kept": kept}


# ---- the work that a pass cannot do without ------------------------------------

def _seen(case):
    """(row, key) pairs that see each other, and the keys that some row sees."""
    rows, keys, window = case["rows"], case["keys"], case["window"]
    if not window:
        return rows * keys - rows * (rows - 1) // 2, keys
    pairs = sum(min(window, keys - rows + i + 1) for i in range(rows))
    return pairs, min(keys, rows + window - 1)


def work(case):
    kind = case["kind"]
    if kind == "append":  # FP32 in, codes and scales out, these in and FP32 out
        return {"bytes": int(2 * case["n"] * case["hd"] * (4 + 2 * 9 / 16 + 4)), "flops": 0}
    if kind == "evict":
        return {"bytes": 4 * case["sets"] * (2 * case["len"] + case["keep"]), "flops": 0}
    pairs, keys = _seen(case)
    hd, heads = case["hd"], case["heads"]
    if kind == "weights":
        return {"bytes": 4 * (keys * hd + case["rows"] * heads * hd + 2 * case["keys"]), "flops": 2 * hd * heads * pairs}
    more = 8 * case["keys"] if case["weights"] else 0
    return {"bytes": keys * hd * 9 // 8 + 8 * case["rows"] * heads * hd + more, "flops": 4 * hd * heads * pairs}


# ---- the same in 64 bits ---------------------------------------------------------

def _exact_values(x):
    """What the cache holds of x, by the format's definition."""
    a = x.double().unflatten(1, (-1, GROUP))
    top = a.abs().max(dim=2, keepdim=True).values
    s = (top / 7).to(torch.float32).to(torch.bfloat16).double()
    s[s == 0] = 1.0
    return (s * torch.clip(torch.round(torch.div(a, s)), -7.0, 7.0)).flatten(1)


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "append":
        return {"k": _exact_values(x["k"]), "v": _exact_values(x["v"])}
    if kind == "evict":
        rows, kept = [], []
        for w in x["w"].double().cpu().numpy():
            mid = np.arange(case["first"], case["len"] - case["recent"])
            best = mid[np.lexsort((mid, -w[mid]))][:case["keep"] - case["first"] - case["recent"]]
            r = np.union1d(best, np.setdiff1d(np.arange(case["len"]), mid))
            rows.append(r)
            kept.append(np.concatenate([w[r], np.zeros(case["len"] - len(r))]))
        return {"rows": np.array(rows), "kept": np.array(kept)}
    rows, keys, window = case["rows"], case["keys"], case["window"]
    quantised = kind == "attn"
    k = _exact_values(x["k"]) if quantised else x["k"].double()
    v = _exact_values(x["v"]) if quantised else None
    got = torch.zeros(keys, dtype=torch.float64, device=k.device)
    y = []
    step = 64  # rows at a time
    for r0 in range(0, rows, step):
        r1 = min(rows, r0 + step)
        lo = max(0, keys - rows + r0 - window + 1) if window else 0
        hi = keys - rows + r1
        q = x["q"][r0:r1].double().transpose(0, 1).flatten(0, 1)  # [heads * rows, hd]
        s = torch.matmul(q, k[lo:hi].T).unflatten(0, (-1, r1 - r0))
        ahead = torch.arange(lo, hi, device=k.device)[None, :] - torch.arange(keys - rows + r0, hi, device=k.device)[:, None]
        hidden = (ahead > 0) | (ahead <= -window) if window else ahead > 0
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        got[lo:hi] += p.sum((0, 1))
        if quantised:
            y.append((p @ v[lo:hi]).transpose(0, 1))
    out = {"y": torch.cat(y)} if quantised else {}
    if "before" in x:
        out["weights"] = x["before"].double() + got
    return out
