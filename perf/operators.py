"""Operators around drafted tokens, as cases that can be timed and checked.

A model that checks several drafted tokens in one pass runs their attention as a
tree over the KV cache, reads the tied head once for all of them, picks a token
per row by probability and keeps the accepted rows of the cache:

  tree     attention of a tree of drafted tokens over a cache
  head     the tied BF16 head for several hidden states, with scale and softcap
  sample   tokens by temperature, top-k, top-p and min-p from given random numbers
  cache    rows of a cache's planes, kept in place or copied into another cache

Sizes are a Gemma-4-E2B-shaped decoder's (8 query heads on one KV head, head dims
256 and 512, a 512-key window, hidden 1536, 262144 tokens, 15 layers with a cache
of their own) or generic ones around them.
"""
import math

import numpy as np
import torch

own = False

HEADS, WINDOW, HIDDEN, VOCAB, SOFTCAP = 8, 512, 1536, 262144, 30.0


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # a chain of a few drafted tokens early in a chat, in a windowed layer
        {"name": "tree_chain", "kind": "tree", "nodes": 4, "heads": HEADS, "hd": 256, "prefix": 203, "window": WINDOW},
        # an ordinary draft tree in a layer that sees everything
        {"name": "tree_draft", "kind": "tree", "nodes": 16, "heads": HEADS, "hd": 512, "prefix": 1900, "window": 0},
        # a wider tree in a windowed layer, far past the window
        {"name": "tree_window", "kind": "tree", "nodes": 37, "heads": HEADS, "hd": 256, "prefix": 2777, "window": WINDOW},
        # a full tree after a long document
        {"name": "tree_long", "kind": "tree", "nodes": 64, "heads": HEADS, "hd": 512, "prefix": 16000, "window": 0},
        # one 4096-row chunk of the vocabulary, as a page that streams the head runs it
        {"name": "head_chunk", "kind": "head", "n": 17, "rows": 4096, "width": HIDDEN},
        # the whole vocabulary for a chain of drafted tokens
        {"name": "head_chain", "kind": "head", "n": 5, "rows": VOCAB, "width": HIDDEN},
        # and for a full tree
        {"name": "head_tree", "kind": "head", "n": 64, "rows": VOCAB, "width": HIDDEN},
        # one token of a chat, with the usual settings
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": VOCAB, "temperature": 1.0, "top_k": 64, "top_p": 0.95, "min_p": 0.0, "spread": 3.0, "ties": False, "banned": 0.0},
        # rows with equal logits (made in 16 bits) and tokens that a grammar forbids
        {"name": "sample_ties", "kind": "sample", "rows": 7, "vocab": 100003, "temperature": 0.7, "top_k": 0, "top_p": 1.0, "min_p": 0.05, "spread": 2.0, "ties": True, "banned": 0.5},
        # a full tree's rows, flat distributions cut by their mass alone
        {"name": "sample_tree", "kind": "sample", "rows": 64, "vocab": VOCAB, "temperature": 0.8, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "spread": 2.0, "ties": False, "banned": 0.0},
        # after a check: five of sixteen appended rows stay, in every plane of 15 layers
        {"name": "cache_keep", "kind": "cache", "n": 5, "of": 16, "at": 1900, "planes256": 24, "planes512": 6, "place": True},
        # a second answer to a long prompt: its cache copied
        {"name": "cache_fork", "kind": "cache", "n": 4000, "of": 4096, "at": 0, "planes256": 24, "planes512": 6, "place": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "head", "sample", "sample", "cache"])
    if kind == "tree":
        return {"kind": kind, "nodes": _log(rng, 1, 64), "heads": rng.choice([1, 2, 3, 4, 6, 8, 8]),
                "hd": rng.choice([64, 128, 256, 256, 512, 512]), "prefix": _log(rng, 1, 16000),
                "window": rng.choice([0, WINDOW, WINDOW, rng.randint(2, 1500)])}
    if kind == "head":
        return {"kind": kind, "n": _log(rng, 2, 64), "rows": _log(rng, 1000, VOCAB),
                "width": rng.choice([HIDDEN, HIDDEN, 8 * rng.randint(32, 192)])}
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 300, VOCAB),
                "temperature": round(rng.uniform(0.4, 1.5), 3),
                "top_k": rng.choice([0, 0, 1, _log(rng, 2, 1000), _log(rng, 2, 1000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3), round(rng.uniform(0.8, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]),
                "spread": round(rng.uniform(1.0, 5.0), 2), "ties": rng.random() < 0.3,
                "banned": rng.choice([0.0, 0.0, round(rng.random(), 2)])}
    if rng.random() < 0.5:
        n = rng.randint(1, 24)
        return {"kind": kind, "n": n, "of": rng.randint(n, 64), "at": _log(rng, 1, 8000),
                "planes256": 2 * rng.randint(1, 12), "planes512": 2 * rng.randint(0, 3), "place": True}
    n = _log(rng, 2, 4000)
    return {"kind": kind, "n": n, "of": rng.randint(n, 4096), "at": rng.randint(0, 96),
            "planes256": 2 * rng.randint(1, 12), "planes512": 2 * rng.randint(0, 3), "place": False}


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
    g.manual_seed(int(seed) * 9973 + 5)
    return g


def _normal(g, *shape, sigma=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * sigma


def _f32(x):
    return float(np.float32(x))


def _tree(nodes, seed):
    """Parents of a draft tree: each node follows one of the few before it, or the prefix."""
    r = np.random.RandomState((int(seed) * 131 + 7) % (1 << 31))
    return [-1 if i == 0 else int(r.randint(max(-1, i - 7), i)) for i in range(nodes)]


def _logits(case, g):
    """Capped logits with a few likely tokens; `ties`: rounded to 16 bits, as a head in
    that type leaves them; `banned`: this share at minus infinity."""
    rows, vocab = case["rows"], case["vocab"]
    x = _normal(g, rows, vocab, sigma=case["spread"])
    likely = torch.randint(0, vocab, (rows, 12), generator=g, device="cuda")
    x.scatter_add_(1, likely, 4.0 * case["spread"] + _normal(g, rows, 12, sigma=1.5))
    x = 30.0 * torch.tanh(x / 30.0)
    if case["ties"]:
        x = x.bfloat16().float()
    if case["banned"]:
        x = x.masked_fill(torch.rand(rows, vocab, generator=g, device="cuda") < case["banned"], -math.inf)
    return x


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "tree":
        # normed rows: q.k of a few units, as trained q and k norms leave it
        hd, keys = case["hd"], case["prefix"] + case["nodes"]
        at = 1.5 / math.sqrt(math.sqrt(hd))
        return {"q": _normal(g, case["nodes"], case["heads"], hd, sigma=at),
                "k": _normal(g, keys, hd, sigma=at), "v": _normal(g, keys, hd),
                "parents": torch.tensor(_tree(case["nodes"], seed), dtype=torch.int32, device="cuda")}
    if kind == "head":
        # normed hidden states and rows of 0.03: logits of about one unit, some capped
        x = _normal(g, case["n"], case["width"])
        x[0] *= 20.0
        return {"x": x, "E": _normal(g, case["rows"], case["width"], sigma=0.03).bfloat16()}
    if kind == "sample":
        return {"x": _logits(case, g), "u": torch.rand(case["rows"], generator=g, device="cuda")}
    cap = case["at"] + case["of"]
    planes = {"c256": _normal(g, case["planes256"], cap, 256)}
    if case["planes512"]:
        planes["c512"] = _normal(g, case["planes512"], cap, 512)
    pick = torch.randperm(case["of"], generator=g, device="cuda")[:case["n"]].sort().values
    planes["rows"] = (pick + case["at"]).to(torch.int32)
    return planes


def prepare(case, seed):
    st = {n: _Held(t) for n, t in _inputs(case, seed).items()}
    st["case"] = case
    kind = case["kind"]
    if kind == "tree":
        st["y"] = _Held(torch.zeros(case["nodes"], case["heads"], case["hd"], device="cuda"))
    elif kind == "head":
        st["y"] = _Held(torch.zeros(case["n"], case["rows"], device="cuda"))
    elif kind == "sample":
        st["tokens"] = _Held(torch.zeros(case["rows"], dtype=torch.int32, device="cuda"))
        st["probs"] = _Held(torch.zeros(case["rows"], device="cuda"))
    else:
        names = [n for n in ("c256", "c512") if n in st]
        to = {n: st[n] if case["place"] else _Held(torch.zeros(st[n].t.shape[0], case["n"], st[n].t.shape[2], device="cuda"))
              for n in names}
        st["to"] = to
        if own:  # the planes of every layer, as a program keeps them
            def planes(of):
                return [of[n].ptr + 4 * i * of[n].t.shape[1] * of[n].t.shape[2]
                        for n in names for i in range(of[n].t.shape[0])]

            st["planes"] = _library().CachePlanes(
                planes(to), planes(st), [st[n].t.shape[2] for n in names for _ in range(st[n].t.shape[0])])
    return st


# ---- one pass ------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    kind = case["kind"]
    if kind == "tree":
        return _attend(case, st["q"].t, st["k"].t, st["v"].t, st["parents"].t)
    if kind == "head":
        return SOFTCAP * torch.tanh((st["x"].t @ st["E"].t.float().T) / SOFTCAP)
    if kind == "sample":
        return _pick(case, st["x"].t, st["u"].t)
    rows = st["rows"].t.long()
    at = case["at"] if case["place"] else 0
    for n, c in st["to"].items():
        c.t[:, at:at + case["n"]] = st[n].t[:, rows]
    return {n: c.t for n, c in st["to"].items()}


def _run_own(st):
    import g4hip
    case = st["case"]
    kind = case["kind"]
    if kind == "tree":
        g4hip.attention_tree(st["q"], st["k"], st["v"], case["nodes"], case["heads"], case["hd"],
                             case["prefix"], st["parents"], case["window"] > 0, case["window"], st["y"])
        return st["y"].t
    if kind == "head":
        g4hip.bf16_head_rows(st["x"], case["n"], st["E"], case["rows"], case["width"], st["y"],
                             scale=1.0, softcap=SOFTCAP)
        return st["y"].t
    if kind == "sample":
        g4hip.sample(st["x"], case["rows"], case["vocab"], st["u"], st["tokens"], st["probs"],
                     temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"],
                     min_p=case["min_p"])
        return {"tokens": st["tokens"].t, "probs": st["probs"].t}
    st["planes"].rows(st["rows"], case["n"], case["at"] if case["place"] else 0,
                      case["at"] + case["of"])
    return {n: c.t for n, c in st["to"].items()}


def _attend(case, q, k, v, parents):
    """softmax(q.k) v, node i seeing the prefix, itself and its ancestors, of these the ones
    within the window of its position (prefix + depth)."""
    nodes, heads, hd, prefix, window = (case[n] for n in ("nodes", "heads", "hd", "prefix", "window"))
    ids = torch.arange(nodes, device=q.device)
    step = (parents.long()[:, None] == ids[None, :]).float()
    eye = torch.eye(nodes, device=q.device)
    # (1 - step)^-1 = 1 + step + step^2 + ...: the ancestors, whole numbers
    above = torch.linalg.solve_triangular(eye - step, eye, upper=False, unitriangular=True)
    depth = above.sum(1).round().long() - 1
    pos = prefix + depth
    sees = torch.cat([torch.ones(nodes, prefix, dtype=torch.bool, device=q.device), above > 0.5], 1)
    if window:
        at = torch.cat([torch.arange(prefix, device=q.device), pos])
        sees = sees & (at[None, :] > pos[:, None] - window)
    s = (q.reshape(nodes * heads, hd) @ k.T).view(nodes, heads, -1)
    s = s.masked_fill(~sees[:, None, :], -math.inf)
    p = torch.exp(s - s.max(-1, keepdim=True).values)
    y = p.view(nodes * heads, -1) @ v
    return y.view(nodes, heads, hd) / p.sum(-1, keepdim=True)


def _pick(case, x, u):
    """One token per row.  In 64 bits: a token's border in the summed probabilities may lie
    next to the random number."""
    vocab, k = case["vocab"], case["top_k"]
    top_p, min_p = _f32(case["top_p"]), _f32(case["min_p"])
    x = torch.where(torch.isfinite(x), x, torch.full_like(x, -math.inf))
    best, order = torch.sort(x, dim=1, descending=True, stable=True)
    d = (best.double() - best[:, :1].double()) / _f32(case["temperature"])
    p = torch.exp(d)
    if 0 < k < vocab:
        p[:, k:] = 0.0
    before = torch.cumsum(p, 1) - p
    keep = p >= min_p
    if top_p < 1.0:
        keep = keep & (before < top_p * p.sum(1, keepdim=True))
    p = torch.where(keep, p, torch.zeros_like(p))
    p = torch.zeros_like(p).scatter_(1, order, p)  # by index again
    upto = torch.cumsum(p, 1)
    total = upto[:, -1:]
    token = (upto <= u.double()[:, None] * total).sum(1, keepdim=True).clamp(max=vocab - 1)
    return {"tokens": token[:, 0].to(torch.int32), "probs": (p.gather(1, token) / total)[:, 0].float()}


# ---- the work that a pass cannot do without ------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "tree":
        n, h, hd, w = case["nodes"], case["heads"], case["hd"], case["window"]
        seen = min(case["prefix"], w - 1) if w else case["prefix"]
        return {"bytes": 4 * hd * (2 * (seen + n) + 2 * n * h) + 4 * n, "flops": 4 * hd * h * n * (seen + 1)}
    if kind == "head":
        n, r, k = case["n"], case["rows"], case["width"]
        return {"bytes": 2 * r * k + 4 * n * (k + r), "flops": 2 * n * r * k}
    if kind == "sample":
        return {"bytes": 4 * case["rows"] * (case["vocab"] + 3), "flops": 0}
    return {"bytes": 8 * case["n"] * (256 * case["planes256"] + 512 * case["planes512"]) + 4 * case["n"],
            "flops": 0}


# ---- the same in 64 bits ---------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "tree":
        return _exact_tree(case, s, _tree(case["nodes"], seed))
    if kind == "head":
        z = torch.matmul(s["x"].double(), s["E"].double().T)
        return torch.tanh(z.div_(SOFTCAP)).mul_(SOFTCAP)
    if kind == "sample":
        return {"tokens": None, "probs": _exact_probs(case, s)}
    out = {}
    for n in ("c256", "c512"):
        if n in s:
            c = s[n].double()
            got = torch.stack([c[:, r] for r in s["rows"].tolist()], 1)
            if case["place"]:
                at = case["at"]
                got = torch.cat([c[:, :at], got, c[:, at + case["n"]:]], 1)
            out[n] = got
    return out


def _exact_tree(case, s, parents):
    q, k, v = (s[n].double() for n in "qkv")
    prefix, window = case["prefix"], case["window"]
    out = []
    for i in range(case["nodes"]):
        path, j = [], i
        while j >= 0:
            path.append(j)
            j = parents[j]
        path.reverse()  # path[d] sits at position prefix + d
        pos = prefix + len(path) - 1
        first = max(0, pos - window + 1) if window else 0
        rows = list(range(first, prefix)) + [prefix + j for d, j in enumerate(path) if prefix + d >= first]
        at = torch.tensor(rows, device=q.device)
        w = torch.softmax(q[i] @ k[at].T, -1)
        out.append(w @ v[at])
    return torch.stack(out)


def _exact_probs(case, s):
    """The picked token's probability among the kept ones, row by row."""
    out = []
    for x, u in zip(s["x"].double(), s["u"].double()):
        ids = torch.nonzero(torch.isfinite(x))[:, 0]
        ids = ids[torch.argsort(x[ids], descending=True, stable=True)]
        if case["top_k"]:
            ids = ids[:case["top_k"]]
        z = x[ids] / _f32(case["temperature"])
        p = torch.softmax(z, 0)
        n = len(ids)
        if case["top_p"] < 1:
            n = min(n, int((torch.cumsum(p, 0) < _f32(case["top_p"])).sum()) + 1)
        n = min(n, int((torch.exp(z - z[0]) >= _f32(case["min_p"])).sum()))
        by_index = ids[:n].sort()
        kept = p[:n][by_index.indices]
        kept = kept / kept.sum()
        at = min(int(torch.searchsorted(torch.cumsum(kept, 0), u, right=True)), n - 1)
        out.append(kept[at])
    return torch.stack(out)
