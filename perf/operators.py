"""Operators of a batch that answers over one shared prompt, each one pass through its public calls.

A case is a dict of plain values.  Its "kind" names the operator:

  product  rows of activations quantized to int8 (one scale a row) times an int8 matrix with one
           scale per output channel, optionally added to a residual: HipRows.quantize + .matmul
  attend   one query row per sequence over a prefix that all sequences share and over the
           sequence's own positions, both int8 caches: HipSharedAttention.run
  choose   penalties for repeated tokens, biases and an allowed-token bitmask on logits, then the
           selected ids with their log-probabilities, or the adjusted logits: HipSelector.run

With `own` false, run() computes the same in elementary torch operations.  Matrices are fixed (a
program serves one model); activations, caches, histories and masks come from the seed.
"""

from __future__ import annotations

import collections
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEVICE = "cuda"
HD = 64  # head dimension of every cache here
LIMIT = 8192 * 4096 * 4096  # multiply-adds of the largest product
ATTEND_LIMIT = 128 * 32 * 33024  # (query head, position) pairs of the largest attention
OWN_LIMIT = 1 << 19  # cache rows (sequence, KV head, position) of the sequences' own positions
LOGIT_LIMIT = 301 * 50001  # logits of the largest selection


def listed():
    return [
        # One token's hidden row through a square projection: latency.
        dict(name="product_1x4096x4096", kind="product", rows=1, n=4096, k=4096, add=False, pad=0),
        # The logits of a decoding batch over the synthetic decoder's vocabulary.
        dict(name="product_64x32768x512", kind="product", rows=64, n=32768, k=512, add=False, pad=0),
        # A prompt's feed-forward down product onto the residual stream, ragged rows, strided input.
        dict(name="product_2001x512x2048_add", kind="product", rows=2001, n=512, k=2048, add=True, pad=64),
        # A large prompt batch through a wide model's projection.
        dict(name="product_8192x4096x4096", kind="product", rows=8192, n=4096, k=4096, add=False, pad=0),
        # The first answer token of a single request: nothing but the prompt and itself.
        dict(name="attend_b1_p512", kind="attend", batch=1, kv_heads=8, rep=1, prefix=512, own=1),
        # The decoding batch of 64 over one 2048-token tool prompt, answers of up to 128 tokens.
        dict(name="attend_b64_p2048", kind="attend", batch=64, kv_heads=8, rep=1, prefix=2048, own=128),
        # Grouped heads, a prompt that ends inside a tile, long ragged answers (some empty).
        dict(name="attend_b33_p4097_gqa", kind="attend", batch=33, kv_heads=4, rep=2, prefix=4097, own=1777),
        # Many requests over one long document.
        dict(name="attend_b128_p32768", kind="attend", batch=128, kv_heads=8, rep=4, prefix=32768, own=256),
        # One constrained answer over the shipped vocabulary.
        dict(name="choose_1x8192", kind="choose", batch=1, vocab=8192, history=640, bias=8, mask=True,
             logits=False),
        # The constrained decoding batch, 2% of the ids allowed, histories of up to 2048 tokens.
        dict(name="choose_64x32768", kind="choose", batch=64, vocab=32768, history=2048, bias=64, mask=True,
             logits=False),
        # A large batch over an odd vocabulary whose adjusted logits a host samples from.
        dict(name="choose_301x50001_logits", kind="choose", batch=301, vocab=50001, history=1000, bias=300,
             mask=True, logits=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "attend", "choose"])
    if kind == "product":
        k = 1 << rng.randint(7, 13)
        rows, n = _log(rng, 1, 8192), _log(rng, 64, 32768)
        n = max(64, min(n, LIMIT // (k * rows), (1 << 26) // max(rows, k)))
        return dict(kind=kind, rows=rows, n=n, k=k, add=rng.random() < 0.3, pad=rng.choice([0, 0, 4, 64]))
    if kind == "attend":
        heads, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8])
        batch = _log(rng, 1, 128)
        mine = min(_log(rng, 1, 2048), max(1, OWN_LIMIT // (batch * heads)))
        most = max(1, ATTEND_LIMIT // (batch * heads * rep) - mine)
        prefix = 0 if rng.random() < 0.05 else min(_log(rng, 16, 32768), most)
        return dict(kind=kind, batch=batch, kv_heads=heads, rep=rep, prefix=prefix, own=mine)
    vocab = _log(rng, 1000, 65000)
    return dict(kind=kind, batch=max(1, min(_log(rng, 1, 301), LOGIT_LIMIT // vocab)), vocab=vocab,
                history=rng.choice([0, _log(rng, 8, 4096), _log(rng, 8, 4096)]),
                bias=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.7,
                logits=rng.random() < 0.4)


# ------------------------------------------------------------------------------- inputs

def _gen(seed, salt):
    return torch.Generator(device=DEVICE).manual_seed(1000003 * salt + seed)


def _normal(seed, salt, *shape):
    return torch.randn(shape, generator=_gen(seed, salt), device=DEVICE, dtype=torch.float32)


def _uniform(seed, salt, lo, hi, *shape):
    return torch.rand(shape, generator=_gen(seed, salt), device=DEVICE, dtype=torch.float32) * (hi - lo) + lo


def _ints(seed, salt, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=_gen(seed, salt), device=DEVICE)


_weights: dict = {}


def _weight(n, k):
    """The model's matrix of this shape: codes [n][k] and one scale per output channel."""
    if (n, k) not in _weights:
        _weights[n, k] = (_ints(n, k, -127, 128, n, k).to(torch.int8), _uniform(k, n, 0.001, 0.02, n))
    return _weights[n, k]


def _lengths(case, seed):
    """Own positions of each sequence: 0 to `own`, evenly spread (the longest always there), in an
    order that the seed gives."""
    b, top = case["batch"], case["own"]
    spread = torch.arange(b, 0, -1, device=DEVICE).mul(top).div(b, rounding_mode="floor")
    if b > 2:
        spread[-1] = 0  # a sequence whose first token is still to be appended
    return spread[torch.randperm(b, generator=_gen(seed, 9), device=DEVICE)]


def _inputs(case, seed):
    kind = case["kind"]
    if kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        x = _normal(seed, 1, rows, k + case["pad"])
        x[:, :: 97] *= 8.0  # channels that stand out, as hidden states have
        return dict(x=x, add=_normal(seed, 2, rows, n) if case["add"] else None)
    if kind == "attend":
        b, h, p, o = (case[f] for f in ("batch", "kv_heads", "prefix", "own"))
        return dict(q=_normal(seed, 1, b, h * case["rep"], HD),
                    prefix_k=_normal(seed, 2, p, h, HD), prefix_v=_normal(seed, 3, p, h, HD),
                    own_k=_normal(seed, 4, o, b * h, HD), own_v=_normal(seed, 5, o, b * h, HD),
                    lengths=_lengths(case, seed))
    b, v, n, c = (case[f] for f in ("batch", "vocab", "history", "bias"))
    zipf = torch.exp(_uniform(seed, 1, 0.0, math.log(v), b, n)).long() - 1  # tokens repeat
    lengths = _ints(seed, 2, (n + 1) // 2, n + 1, b)
    words = (v + 31) // 32
    allowed = _uniform(seed, 3, 0.0, 1.0, b, words * 32) < 0.02
    allowed[:, v:] = False
    allowed[torch.arange(b, device=DEVICE), _ints(seed, 4, 0, v, b)] = True
    if b > 2:
        allowed[seed % b] = False  # a grammar at a dead end
    bits = (allowed.view(b, words, 32).long() << torch.arange(32, device=DEVICE)).sum(-1)
    return dict(logits=_normal(seed, 5, b, v) * 4, history=zipf.clamp(0, v - 1).int(), lengths=lengths.int(),
                prompt=(lengths // 2).int(), repetition=_uniform(seed, 6, 1.0, 1.5, b),
                presence=_uniform(seed, 7, 0.0, 1.0, b), frequency=_uniform(seed, 8, 0.0, 0.5, b),
                bias_ids=_ints(seed, 9, 0, v, b, c).int(), bias=_normal(seed, 10, b, c) * 4,
                bias_counts=_ints(seed, 11, (c + 1) // 2, c + 1, b).int(),
                mask=torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int() if case["mask"] else None)


# ------------------------------------------------------------------------------ prepare

class _State:
    """What the program holds."""

    def __init__(self, case, **held):
        self.case = case
        self.__dict__.update(held)

    def __del__(self):
        for handle in getattr(self, "handles", ()):
            handle.free()


_program: dict = {}
_recent: collections.deque = collections.deque(maxlen=4)  # states whose buffers were handed out


def _backend():
    if "hip" not in _program:
        root = Path(__file__).resolve().parent.parent
        if str(root / "needle.js_amd") not in sys.path:
            sys.path.insert(0, str(root / "needle.js_amd"))
        import needle_hip

        _program["lib"] = needle_hip
        _program["hip"] = needle_hip.HipBackend(device=0)
    return _program["hip"]


def _matrix(n, k):
    """The matrix in HBM, uploaded once."""
    if ("mat", n, k) not in _program:
        w, s = _weight(n, k)
        _program["mat", n, k] = _backend().upload(
            _program["lib"].Int8Matrix(w.cpu().numpy(), s.cpu().numpy().reshape(n, 1), k))
    return _program["mat", n, k]


def _quantized(x):
    """Codes and scales of rows [..., HD] as the cache holds them: m = max(1e-12, max|x|) and
    s = m / 127 in 64 bits, code = x / s rounded to the nearest, ties to even."""
    s = x.abs().amax(-1).double().clamp_min(1e-12) / 127
    return torch.round(x.double() / s[..., None]).to(torch.int8), s.float()


def prepare(case, seed):
    kind, data = case["kind"], _inputs(case, seed)
    if kind == "product":
        data["w"], data["sw"] = _weight(case["n"], case["k"])
    if kind == "attend":
        h = case["kv_heads"]
        for part, heads in (("prefix", (h,)), ("own", (case["batch"], h))):
            for kv in "kv":
                codes, scales = _quantized(data[f"{part}_{kv}"])
                data[f"{part}_{kv}c"] = codes.movedim(0, -2).reshape(heads + (-1, HD)).contiguous()
                data[f"{part}_{kv}s"] = scales.movedim(0, -1).reshape(heads + (-1,)).contiguous()
    if own:
        _adopt(case, data)
    for name in ("prefix_k", "prefix_v", "own_k", "own_v"):
        data.pop(name, None)
    state = _State(case, **data)
    _recent.append(state)
    return state


def _adopt(case, data):
    """The program's handles: caches filled position by position, workspaces, output buffers."""
    hip, kind = _backend(), case["kind"]
    nh = _program["lib"]
    if kind == "product":
        data["mat"] = _matrix(case["n"], case["k"])
        data["rows"] = nh.HipRows(hip, case["rows"], case["k"])
        data["y"] = torch.empty((case["rows"], case["n"]), device=DEVICE)
        data["handles"] = [data["rows"]]
    elif kind == "attend":
        b, h, hq = case["batch"], case["kv_heads"], case["kv_heads"] * case["rep"]
        prefix = nh.HipKvCache(hip, 1, h, max(1, case["prefix"]))
        mine = nh.HipKvCache(hip, 1, b * h, case["own"])
        torch.cuda.synchronize()
        for cache, name, count in ((prefix, "prefix", case["prefix"]), (mine, "own", case["own"])):
            hip._check(hip.lib.nd_kv_store_d(hip.ctx, cache.handle, 0, 0, count,
                                             data[name + "_k"].data_ptr(), data[name + "_v"].data_ptr(), None))
        hip._check(hip.lib.nd_sync(hip.ctx))
        data["lengths32"] = data["lengths"].int()
        data["out"] = torch.empty((b, hq, HD), device=DEVICE)
        data["shared"] = nh.HipSharedAttention(hip, b, h, hq)
        data["prefix"], data["mine"] = prefix, mine
        data["handles"] = [data["shared"], prefix, mine]
    else:
        b, v = case["batch"], case["vocab"]
        data["selector"] = nh.HipSelector(hip, b)
        adjust = nh.LogitAdjust()
        for name in ("repetition", "presence", "frequency"):
            setattr(adjust, name, data[name].data_ptr())
        if case["history"]:
            adjust.history, adjust.history_stride = data["history"].data_ptr(), case["history"]
            adjust.history_lengths = data["lengths"].data_ptr()
            adjust.prompt_lengths = data["prompt"].data_ptr()
        if case["bias"]:
            adjust.bias_ids, adjust.bias = data["bias_ids"].data_ptr(), data["bias"].data_ptr()
            adjust.bias_stride, adjust.bias_counts = case["bias"], data["bias_counts"].data_ptr()
        data["adjust"] = adjust
        data["ids"] = torch.empty(b, dtype=torch.int32, device=DEVICE)
        data["lps"] = torch.empty(b, dtype=torch.float64, device=DEVICE)
        data["out"] = torch.empty((b, v), device=DEVICE) if case["logits"] else None
        data["handles"] = [data["selector"]]


# ---------------------------------------------------------------------------------- run

def run(state):
    case, kind = state.case, state.case["kind"]
    if own:
        if kind == "product":
            state.rows.quantize(state.x.data_ptr(), case["rows"], case["k"] + case["pad"])
            state.rows.matmul(state.mat, state.y.data_ptr(),
                              add=None if state.add is None else state.add.data_ptr())
            return {"y": state.y}
        if kind == "attend":
            state.shared.run(state.prefix, case["prefix"], state.mine, state.lengths32.data_ptr(),
                             case["own"], 0, state.q.data_ptr(), state.out.data_ptr())
            return {"out": state.out}
        state.selector.run(state.logits.data_ptr(), case["batch"], case["vocab"], state.ids.data_ptr(),
                           state.lps.data_ptr(), adjust=state.adjust,
                           mask=None if state.mask is None else state.mask.data_ptr(),
                           out=None if state.out is None else state.out.data_ptr())
        picked = {"ids": state.ids, "log_probabilities": state.lps}
        return picked if state.out is None else {**picked, "logits": state.out}
    if kind == "product":
        return _product(state)
    return _attend(state) if kind == "attend" else _choose(state)


def _product(s):
    x = s.x[:, : s.case["k"]]
    codes, sx = _quantized(x)  # in 64 bits: codes next to a border
    y = torch.matmul(codes.float(), s.w.float().t()) * s.sw[None, :] * sx[:, None]
    return {"y": y if s.add is None else s.add + y}


def _attend(s):
    case = s.case
    b, h, rep, p, o = (case[f] for f in ("batch", "kv_heads", "rep", "prefix", "own"))
    q = s.q.view(b, h, rep, HD)
    # Scores of the shared positions for all sequences' rows together, then of each one's own.
    shared = torch.matmul(q.transpose(0, 1).reshape(h, b * rep, HD), s.prefix_kc.float().transpose(1, 2))
    shared = (shared * (s.prefix_ks[:, None, :] * 0.125)).view(h, b, rep, p).transpose(0, 1)
    mine = torch.matmul(q, s.own_kc.float().transpose(2, 3)) * (s.own_ks[:, :, None, :] * 0.125)
    seen = torch.arange(o, device=DEVICE)[None, :] < s.lengths[:, None]
    mine = mine.masked_fill(~seen[:, None, None, :], -math.inf)
    scores = torch.cat([shared, mine], dim=-1)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    e = torch.where(total > 0, e / total, 0.0)
    ep = e[..., :p].transpose(0, 1).reshape(h, b * rep, p) * s.prefix_vs[:, None, :]
    out = torch.matmul(ep, s.prefix_vc.float()).view(h, b, rep, HD).transpose(0, 1)
    out = out + torch.matmul(e[..., p:] * s.own_vs[:, :, None, :], s.own_vc.float())
    return {"out": out.reshape(b, h * rep, HD)}


def _choose(s):
    case = s.case
    b, v, n, c = (case[f] for f in ("batch", "vocab", "history", "bias"))
    # The adjusted logit is one float32 rounding of the exact expression.
    l = s.logits.double()
    if n:
        at = torch.arange(n, device=DEVICE)[None, :]
        inside = at < s.lengths[:, None]
        ones = inside.float()
        seen = torch.zeros((b, v), device=DEVICE).scatter_add_(1, s.history.long(), ones)
        made = torch.zeros((b, v), device=DEVICE).scatter_add_(
            1, s.history.long(), ones * (at >= s.prompt[:, None]))
        r = s.repetition.double()[:, None]
        l = torch.where(seen > 0, torch.where(l > 0, l / r, l * r), l)
        l = l - s.frequency.double()[:, None] * made - s.presence.double()[:, None] * (made > 0)
    if c:
        entry = torch.arange(1, c + 1, device=DEVICE)[None, :]
        entry = torch.where(entry <= s.bias_counts[:, None], entry, 0)
        last = torch.zeros((b, v), dtype=torch.long, device=DEVICE).scatter_reduce_(
            1, s.bias_ids.long(), entry, "amax")  # the last entry of an id counts
        l = l + torch.where(last > 0, s.bias.double().gather(1, (last - 1).clamp_min(0)), 0.0)
    l = l.float()
    allowed = torch.ones((b, v), dtype=torch.bool, device=DEVICE)
    if s.mask is not None:
        ids = torch.arange(v, device=DEVICE)
        allowed = ((s.mask[:, ids >> 5] >> (ids & 31)) & 1).bool()
    masked = l.masked_fill(~allowed, -math.inf)
    some = allowed.any(1)
    top = masked.amax(1, keepdim=True)
    ids = ((masked == top) & allowed).to(torch.uint8).argmax(1)
    high = l.amax(1).double()
    lp = l.gather(1, ids[:, None])[:, 0].double() - high - torch.log(
        torch.exp(l.double() - high[:, None]).sum(1))
    out = {"ids": torch.where(some, ids, -1).int(), "log_probabilities": torch.where(some, lp, math.nan)}
    return {**out, "logits": masked} if case["logits"] else out


# -------------------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "product":
        m, n, k = case["rows"], case["n"], case["k"]
        moved = 4 * m * k + n * k + 4 * n + 4 * m * n * (2 if case["add"] else 1)
        return {"bytes": moved, "flops": 2 * m * n * k}
    if kind == "attend":
        b, h, rep, p = (case[f] for f in ("batch", "kv_heads", "rep", "prefix"))
        lengths = [case["own"] * i // b for i in range(b, 0, -1)]
        mine = sum(lengths) - (lengths[-1] if b > 2 else 0)
        return {"bytes": 136 * h * (p + mine) + 8 * b * h * rep * HD + 4 * b,
                "flops": 4 * HD * h * rep * (b * p + mine)}
    b, v, n, c = (case[f] for f in ("batch", "vocab", "history", "bias"))
    moved = 4 * b * v * (2 if case["logits"] else 1) + (b * v // 8 if case["mask"] else 0)
    return {"bytes": moved + 3 * b * n + 6 * b * c + 24 * b, "flops": 4 * b * v}


# ------------------------------------------------------------------------------- exact

def exact(case, seed):
    """The operators' definitions, a row or head at a time, in 64 bits."""
    data, kind = _inputs(case, seed), case["kind"]
    if kind == "product":
        w, sw = (t.double() for t in _weight(case["n"], case["k"]))
        x = data["x"][:, : case["k"]].double()
        step = torch.maximum(x.abs().max(1).values, torch.tensor(1e-12, device=DEVICE, dtype=torch.float64)) / 127
        y = torch.round(x / step[:, None]) @ w.T
        y = y * step.float().double()[:, None] * sw
        return {"y": y if data["add"] is None else y + data["add"].double()}
    if kind == "attend":
        return {"out": _exact_attend(case, data)}
    return _exact_choose(case, {k: None if v is None else v.cpu().numpy() for k, v in data.items()})


def _exact_attend(case, data):
    b, h, rep, p = (case[f] for f in ("batch", "kv_heads", "rep", "prefix"))

    def held(x):  # what a cache stands for: code times scale
        step = x.double().abs().amax(-1, keepdim=True).clamp_min(1e-12) / 127
        return torch.round(x.double() / step) * step.float().double()

    out = torch.zeros((b, h * rep, HD), dtype=torch.float64, device=DEVICE)
    q, lengths = data["q"].double(), data["lengths"].tolist()
    for g in range(h):
        pk, pv = held(data["prefix_k"][:, g]), held(data["prefix_v"][:, g])
        for i in range(b):
            n = lengths[i]
            if p + n == 0:
                continue
            k = torch.cat([pk, held(data["own_k"][:n, i * h + g])])
            v = torch.cat([pv, held(data["own_v"][:n, i * h + g])])
            heads = slice(g * rep, (g + 1) * rep)
            out[i, heads] = torch.softmax(q[i, heads] @ k.T / math.sqrt(HD), -1) @ v
    return out


def _exact_choose(case, d):
    b, v = case["batch"], case["vocab"]
    ids, lps, logits = [], [], []
    for r in range(b):
        l = d["logits"][r].astype(np.float64)
        told = d["history"][r][: d["lengths"][r]]
        tokens = np.unique(told)
        pen = float(d["repetition"][r])
        l[tokens] = np.where(l[tokens] > 0, l[tokens] / pen, l[tokens] * pen)
        made, counts = np.unique(told[d["prompt"][r]:], return_counts=True)
        l[made] -= float(d["frequency"][r]) * counts
        l[made] -= float(d["presence"][r])
        table = dict(zip(d["bias_ids"][r][: d["bias_counts"][r]].tolist(), d["bias"][r].tolist()))
        for token, value in table.items():
            l[token] += value
        l = l.astype(np.float32)  # the adjusted logits are float32 values
        if d["mask"] is None:
            ok = np.ones(v, bool)
        else:
            ok = np.unpackbits(d["mask"][r].view(np.uint8), bitorder="little")[:v].astype(bool)
        wide = l.astype(np.float64)
        only = np.where(ok, wide, -np.inf)
        pick = int(np.argmax(only)) if ok.any() else -1
        ids.append(pick)
        top = wide.max()
        lps.append(wide[pick] - top - math.log(np.exp(wide - top).sum()) if ok.any() else math.nan)
        logits.append(only)
    out = {"ids": np.array(ids, np.int32), "log_probabilities": np.array(lps)}
    return {**out, "logits": np.array(logits)} if case["logits"] else out
