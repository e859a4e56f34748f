"""Performance cases of the packed-batch operators.

A packed batch lays the documents of a request batch end to end, [T, ...] with
T the sum of their lengths, instead of padding each to the longest.  Its
operators, and the ones that serve many fine-tunes beside one encoder:

- pack:  the plan of a packed batch from the documents' lengths on the GPU
         (offsets, document and position of every token, slot maps into the
         padded layout), and rows moved into it or back out of it;
- rope:  rotary positions given per token, on one axis or several;
- attn:  attention inside each document: everything, a window, causal, a prefix
         seen by all, scores capped by a tanh, a bias that falls with distance;
         whole documents, chunks of new tokens and single tokens over longer
         keys, grouped heads;
- lora:  a projection with the low-rank adapter of each row's own request
         beside it, on plain and on quantized weights.

Shapes are the ModernBERT-base (hidden 768, 12 heads) and ModernBERT-large
(hidden 1024, 16 heads) ones, with head dimension 64.  `own` selects the
framework's kernels; otherwise run() computes the same in elementary torch
operations.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HEAD = 64       # head dimension
WINDOW = 128    # the encoder's sliding window: keys within 64 of a query
GROUP = 64      # group size of the quantized format
BASE = 10000.0  # the sliding layers' rotation base
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# (in, out) of the encoder's linear layers: Wqkv, attention Wo, Wi, feed-forward Wo
LAYERS = [(768, 2304), (768, 768), (1152, 768), (1024, 1024), (1024, 5248), (2624, 1024)]


# ------------------------------------------------------------------ the cases

def listed():
    """The listed cases, each with the use it stands for."""
    return [
        # a few short prompts of one request batch, packed before the first layer: latency
        {"name": "pack_f32_b4", "op": "pack", "dir": "pack", "t": "f32", "B": 4, "L": 128, "hidden": 768, "empty": 0},
        # a large serving batch handed back padded, as the decision head reads it
        {"name": "unpack_f16_b64_l1024", "op": "pack", "dir": "unpack", "t": "f16", "B": 64, "L": 1024,
         "hidden": 1024, "empty": 1},
        # one prompt in the loaders' default type
        {"name": "rope_f32_t93", "op": "rope", "t": "f32", "T": 93, "heads": 12, "axes": 1, "far": 512},
        # boards and page layouts as tokens with a time, a row and a column, a long packed batch
        {"name": "rope_bf16_t32768_axes", "op": "rope", "t": "bf16", "T": 32768, "heads": 16, "axes": 3, "far": 8192},
        # three prompts of odd lengths through a sliding layer, the loaders' default type
        {"name": "attn_f32_b3_l333_window", "op": "attn", "t": "f32", "B": 3, "L": 333, "new": 0, "heads": 12,
         "kv": 12, "mask": "window", "cap": 0.0, "slopes": False, "empty": 0},
        # a global layer over a ragged serving batch at the default maximum length
        {"name": "attn_f16_b32_l512_full", "op": "attn", "t": "f16", "B": 32, "L": 512, "new": 0, "heads": 12,
         "kv": 12, "mask": "full", "cap": 0.0, "slopes": False, "empty": 0},
        # long documents in a sliding layer whose heads weigh distance
        {"name": "attn_bf16_b8_l4096_bias", "op": "attn", "t": "bf16", "B": 8, "L": 4096, "new": 0, "heads": 16,
         "kv": 16, "mask": "window", "cap": 0.0, "slopes": True, "empty": 0},
        # one new token of each of 48 requests over its own keys, grouped heads, capped scores
        {"name": "attn_bf16_b48_l4096_token", "op": "attn", "t": "bf16", "B": 48, "L": 4096, "new": 1, "heads": 16,
         "kv": 4, "mask": "causal", "cap": 30.0, "slopes": False, "empty": 0},
        # chunks of new tokens of long documents behind a prefix that everybody sees
        {"name": "attn_f16_b4_l8192_chunk", "op": "attn", "t": "f16", "B": 4, "L": 8192, "new": 1000, "heads": 12,
         "kv": 12, "mask": "prefix", "cap": 50.0, "slopes": False, "empty": 0},
        # one row of each of 48 requests, two requests to an adapter: the q / k / v projection
        {"name": "lora_f16_m48_r16", "op": "lora", "t": "f16", "w": "f16", "B": 48, "L": 1, "K": 768, "N": 2304,
         "n": 24, "R": 16, "bias": False},
        # a quantized checkpoint with small adapters on a batch of prompts
        {"name": "lora_q4_b8_l384_r8", "op": "lora", "t": "f16", "w": "q4", "B": 8, "L": 384, "K": 1152, "N": 768,
         "n": 4, "R": 8, "bias": False},
        # a large packed batch of a dozen fine-tunes through the large shape's widest projection
        {"name": "lora_bf16_b32_l900_r64", "op": "lora", "t": "bf16", "w": "bf16", "B": 32, "L": 900, "K": 1024,
         "N": 5248, "n": 12, "R": 64, "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["pack", "rope", "attn", "attn", "attn", "lora", "lora"])
    t = rng.choice(["f16", "bf16", "f32"])
    if op == "pack":
        L = _log(rng, 8, 2048)
        return {"op": op, "dir": rng.choice(["pack", "unpack"]), "t": t, "B": _log(rng, 1, max(2, min(512, 32768 // L))),
                "L": L, "hidden": rng.choice([768, 1024]), "empty": rng.choice([0, 0, 1])}
    if op == "rope":
        return {"op": op, "t": t, "T": _log(rng, 1, 16384), "heads": rng.choice([12, 16]),
                "axes": rng.choice([1, 1, 2, 3]), "far": rng.choice([512, 8192, 131072])}
    if op == "attn":
        heads, kv = rng.choice([(12, 12), (16, 16), (16, 4), (12, 4)])
        mask = rng.choice(["full", "window", "causal", "prefix"])
        L = _log(rng, 16, 2048 if t == "f32" else 4096)
        new = rng.choice([0, 0, 1, _log(rng, 2, max(3, L // 2))])
        pairs = (3 if t == "f32" else 10) * 10 ** 8  # of scores over all heads
        B = _log(rng, 1, max(2, min(64, pairs // (heads * L * (new or L)))))
        return {"op": op, "t": t, "B": B, "L": L, "new": new, "heads": heads, "kv": kv, "mask": mask,
                "cap": rng.choice([0.0, 0.0, 30.0]), "slopes": rng.random() < 0.3, "empty": rng.choice([0, 0, 1])}
    K, N = rng.choice(LAYERS)
    w = rng.choice(["f16", "bf16", "f32", "q8", "q4"])
    t = w if w in TYPES else "f16"
    L = _log(rng, 1, 1024)
    most = 4096 if t == "f32" else 16384
    return {"op": op, "t": t, "w": w, "B": _log(rng, 1, max(2, min(64, most // L))), "L": L, "K": K, "N": N,
            "n": _log(rng, 1, 32), "R": rng.choice([4, 8, 16, 32, 64]), "bias": rng.random() < 0.3}


# ------------------------------------------------------------------ sizes

def _lengths(case):
    """The documents' lengths: spread evenly from an eighth of L to L, as a batch
    of mixed prompts is, after `empty` empty ones."""
    B, L = case["B"], case["L"]
    lo = max(1, L // 8)
    lens = [lo + int((L - lo) * (i + 1) / B) for i in range(B)]
    for i in range(min(case.get("empty", 0), B - 1)):
        lens[i] = 0
    return lens


def _queries(case):
    """Each document's queries: all its tokens, or its last `new` ones."""
    return [min(n, case["new"] or n) for n in _lengths(case)]


def _prefix(case):
    return case["L"] // 16 + 1 if case["mask"] == "prefix" else 0


def _seen(case):
    """(query, key) pairs within the masks, of one head."""
    total = 0
    for n, m in zip(_lengths(case), _queries(case)):
        p = np.arange(n - m, n)
        if case["mask"] == "full":
            seen = np.full(m, n)
        elif case["mask"] == "window":
            seen = np.minimum(p + WINDOW // 2, n - 1) - np.maximum(p - WINDOW // 2, 0) + 1
        else:
            seen = np.maximum(p + 1, min(_prefix(case), n))
        total += int(seen.sum())
    return total


_WBYTES = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8": 1.0 + 2.0 / GROUP, "q4": 0.5 + 4.0 / GROUP}


def work(case):
    es, op = BYTES[case["t"]], case["op"]
    if op == "rope":
        n = case["T"] * 2 * case["heads"] * HEAD
        return {"bytes": 2.0 * n * es + 4 * case["axes"] * case["T"], "flops": 3.0 * n}
    T = sum(_lengths(case))
    if op == "pack":
        rows = T + (T if case["dir"] == "pack" else case["B"] * case["L"])
        return {"bytes": float(rows * case["hidden"] * es + 4 * case["B"] + 4 * (case["B"] + 1) + 12 * T),
                "flops": float(T)}
    if op == "attn":
        Tq = sum(_queries(case))
        return {"bytes": float((2 * Tq * case["heads"] + 2 * T * case["kv"]) * HEAD * es),
                "flops": 4.0 * _seen(case) * HEAD * case["heads"]}
    K, N, R = case["K"], case["N"], case["R"]
    used = min(case["n"], case["B"])
    return {"bytes": T * (K + N) * es + K * N * _WBYTES[case["w"]] + used * R * (K + N) * es + 4.0 * T,
            "flops": 2.0 * T * (K * N + R * (K + N))}


# ------------------------------------------------------------------ inputs

class _Gen:
    """Values from a seed alone, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1000003 * int(seed) + 29)

    def normal(self, shape, std, t):
        return (torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32) * std).to(TYPES[t])

    def ints(self, lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def shuffled(self, values):
        order = torch.randperm(len(values), generator=self.g, device="cuda").tolist()
        return [values[i] for i in order], order


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """Everything a case computes with, as torch tensors made from the seed."""
    g, op, t = _Gen(seed), case["op"], case["t"]
    if op == "rope":
        T, A, H = case["T"], case["axes"], case["heads"]
        # the q / k / v projection's heads side by side; q and k are rotated
        return {"qkv": g.normal((T, 3 * H, HEAD), 1.0, t), "positions": g.ints(0, case["far"], (A, T))}
    lens, order = g.shuffled(_lengths(case))
    T, d = sum(lens), {"lens": lens, "lengths": _i32(lens)}
    if op == "pack":
        d["x"] = g.normal((case["B"], case["L"], case["hidden"]) if case["dir"] == "pack" else (T, case["hidden"]), 1.0, t)
    elif op == "attn":
        new = [_queries(case)[i] for i in order]
        d["new"], d["newLengths"] = new, _i32(new)
        # scores of a trained head reach well past 10
        d["q"] = g.normal((sum(new), case["heads"], HEAD), 2.0, t)
        d["k"], d["v"] = (g.normal((T, case["kv"], HEAD), 1.0, t) for _ in range(2))
        if case["mask"] == "prefix":
            d["prefix"] = _i32([min(_prefix(case), n) for n in lens])
        if case["slopes"]:  # a geometric series over the heads, as distance biases are trained with
            d["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])],
                                       dtype=torch.float32, device="cuda")
    else:
        K, N, R, n, w = case["K"], case["N"], case["R"], case["n"], case["w"]
        d["x"] = g.normal((T, K), 1.0, t)
        if w in TYPES:
            d["w"] = g.normal((N, K), 0.02, w)
        elif w == "q8":  # symmetric codes, about 0.02 in weight
            d["codes"] = (torch.randn((N, K), generator=g.g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8)
            d["scales"] = (0.0005 * (1 + 0.2 * torch.rand((N, K // GROUP), generator=g.g, device="cuda"))).half()
        else:  # affine codes, two to a byte, the even column in the low half
            c = (torch.randn((N, K), generator=g.g, device="cuda") * 2.5 + 7.5).round().clamp(0, 15).to(torch.uint8)
            d["codes"] = c[:, 0::2] | (c[:, 1::2] << 4)
            d["scales"] = (0.008 * (1 + 0.2 * torch.rand((N, K // GROUP), generator=g.g, device="cuda"))).half()
            d["zeros"] = (-7.5 * d["scales"].float()).half()
        d["a"], d["b"] = g.normal((n, R, K), K ** -0.5, t), g.normal((n, N, R), 0.02, t)
        d["alpha"] = torch.full((n,), 2.0, device="cuda")
        # a request's rows share its adapter; some requests have none
        which = g.ints(-1, n, (case["B"],)) if case["B"] > 1 else g.ints(0, n, (1,))
        d["index"] = torch.repeat_interleave(which, d["lengths"].long(), output_size=T)
        d["bias"] = g.normal((N,), 0.1, t) if case["bias"] else None
    return d


def _sections(case):
    """Rotation pairs of each axis."""
    half = HEAD // 2
    return {1: (half,), 2: (half // 2, half // 2), 3: (8, 12, 12)}[case["axes"]]


class _State:
    def __init__(self, case, d):
        self.case, self.d = case, d
        self.calls = None


def prepare(case, seed):
    """The inputs, and for the framework's kernels its handles of them and the
    plans and weights that a program keeps."""
    state = _State(case, _inputs(case, seed))
    if own:
        state.calls = _Calls(case, state.d)
    return state


def run(state):
    if own:
        return state.calls.run()
    return _PLAIN[state.case["op"]](state.case, state.d)


# ------------------------------------------------------------------ the framework's kernels

_shared = {}


def _backend():
    if "be" not in _shared:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "laya-js_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        from laya_hip.backend import HipBackend
        _shared["be"] = HipBackend(0)
    return _shared["be"]


class _Address:
    def __init__(self, ptr, shape, code):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": code, "data": (ptr, False), "version": 2,
                                         "strides": None}


class _Calls:
    """A program's calls on one set of inputs: the tensors uploaded, the plan and
    the weights laid out, the last outputs kept until the next call."""

    def __init__(self, case, d):
        self.be, self.case, self.kept, self.outs, self.views = _backend(), case, [], [], {}
        be, op = self.be, case["op"]
        t = {k: self.keep(be.fromHost(self.host(v))) for k, v in d.items() if isinstance(v, torch.Tensor)}
        if op == "pack":
            total, L = sum(d["lens"]), case["L"]
            if case["dir"] == "pack":
                self.fn = lambda: self.packed(be.packDocs(t["lengths"], total, L), lambda p: be.packRows(t["x"], p))
            else:
                self.fn = lambda: self.packed(be.packDocs(t["lengths"], total, L), lambda p: be.unpackRows(t["x"], p))
        elif op == "rope":
            T, H = case["T"], case["heads"]
            qk = self.keep(be.slice(t["qkv"], [0, 0, 0], [T, 2 * H, HEAD]))
            self.fn = lambda: {"qk": be.ropeAt(qk, t["positions"], BASE, _sections(case))}
        elif op == "attn":
            keys = self.keep(be.packDocs(t["lengths"], sum(d["lens"]), 0))
            docs = self.keep(be.packDocs(t["newLengths"], sum(d["new"]), 0)) if case["new"] else keys
            kind = case["mask"]
            opts = {"keys": keys, "causal": kind in ("causal", "prefix"), "window": WINDOW if kind == "window" else None,
                    "prefix": t.get("prefix"), "cap": case["cap"] or None, "slopes": t.get("slopes")}
            self.fn = lambda: {"o": be.sdpaPacked(t["q"], t["k"], t["v"], docs, HEAD ** -0.5, **opts)}
        else:
            bank = self.keep(be.loraBank(t["a"], t["b"], t["alpha"]))
            from laya_hip.compose import lora_linear_any
            w = t["w"] if "w" in t else self.keep_quantized(d)
            self.fn = lambda: {"y": lora_linear_any(be, t["x"], w, bank, t["index"], t.get("bias"))}
        be.flush()

    def packed(self, p, rows):
        return {"offsets": p.offsets, "doc": p.doc, "pos": p.pos, "slots": p.slots, "rows": rows(p)}

    def keep(self, v):
        self.kept.append(v)
        return v

    def keep_quantized(self, d):
        from laya_hip.host import HostQuantized
        bits = 8 if d["codes"].dtype == torch.int8 else 4
        N, K = d["codes"].shape[0], d["codes"].shape[1] * 8 // bits
        h = HostQuantized((N, K), bits, GROUP, "symmetric" if bits == 8 else "affine",
                          d["codes"].cpu().numpy().view(np.uint8).reshape(-1), self.host(d["scales"]),
                          self.host(d["zeros"]) if "zeros" in d else None)
        q = self.be.fromHostQuantized(h, "f16")
        self.kept += [x for x in (q.w, q.scales, q.biases) if x is not None]
        return q

    @staticmethod
    def host(t):
        from laya_hip.host import HostTensor
        name = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "i32",
                torch.int8: "i8", torch.uint8: "u8"}[t.dtype]
        a = t.contiguous().cpu()
        return HostTensor(name, tuple(t.shape), a.view(torch.int16).numpy().view(np.uint16) if name == "bf16" else a.numpy())

    def view(self, t):
        """A torch tensor over a device tensor's memory."""
        key = (self.be._ptr(t), t.shape, t.dtype)
        if key not in self.views:
            code = {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i32": "<i4"}[t.dtype]
            r = torch.as_tensor(_Address(key[0], t.shape, code), device="cuda")
            self.views[key] = r.view(torch.bfloat16) if t.dtype == "bf16" else r
        return self.views[key]

    def run(self):
        for t in self.outs:
            self.be.dispose(t)
        got = self.fn()
        self.outs = list(got.values())
        return {k: self.view(v) for k, v in got.items()}

    def __del__(self):
        self.be.flush()
        for v in self.outs + self.kept:
            v.dispose() if hasattr(v, "dispose") else self.be.dispose(v)


# ------------------------------------------------------------------ plain forms

def _plan(lengths, total):
    """Offsets [B + 1], and every packed row's document and position."""
    offsets = torch.cat([lengths.new_zeros(1), torch.cumsum(lengths, 0, dtype=torch.int32)])
    doc = torch.repeat_interleave(torch.arange(lengths.numel(), dtype=torch.int32, device=lengths.device), lengths.long(),
                                  output_size=total)
    pos = torch.arange(total, dtype=torch.int32, device=lengths.device) - offsets[doc.long()]
    return offsets, doc, pos


def _plain_pack(case, d):
    offsets, doc, pos = _plan(d["lengths"], sum(d["lens"]))
    slots = doc * case["L"] + pos
    if case["dir"] == "pack":
        rows = d["x"].reshape(-1, case["hidden"])[slots.long()]
    else:
        rows = d["x"].new_zeros(case["B"] * case["L"], case["hidden"])
        rows[slots.long()] = d["x"]
        rows = rows.reshape(case["B"], case["L"], case["hidden"])
    return {"offsets": offsets, "doc": doc, "pos": pos, "slots": slots, "rows": rows}


def _frequencies():
    """Angle per position of each rotation pair, by the contract's rule: rounded
    to 32 bits at each step."""
    half = HEAD // 2
    frac = (np.arange(half) / half).astype(np.float32).astype(np.float64)
    power = (-frac * float(np.float32(math.log2(BASE)))).astype(np.float32).astype(np.float64)
    return np.exp2(power).astype(np.float32)


def _plain_rope(case, d):
    half, dev = HEAD // 2, d["qkv"].device
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=dev), torch.tensor(_sections(case), device=dev),
                                   output_size=half)
    # the angle's product rounds to 32 bits (the contract's rule); its cosine and sine are taken in 64
    angle = (d["positions"].double()[axis].t() * torch.from_numpy(_frequencies()).to(dev).double()).float().double()
    c, s = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    x = d["qkv"][:, :2 * case["heads"]].float()
    a, b = x[..., :half], x[..., half:]
    return {"qk": torch.cat([a * c - b * s, b * c + a * s], -1).to(TYPES[case["t"]])}


def _plain_attn(case, d):
    t, H, KV = TYPES[case["t"]], case["heads"], case["kv"]
    B, Lq, Lk, dev = case["B"], max(d["new"]), max(d["lens"]), d["q"].device
    qoff, qdoc, qpos = _plan(d["newLengths"], sum(d["new"]))
    koff = torch.cat([d["lengths"].new_zeros(1), torch.cumsum(d["lengths"], 0, dtype=torch.int32)])
    i, j = (torch.arange(n, device=dev) for n in (Lq, Lk))
    # padded operands, [B, KV, H / KV * Lq or Lk, 64]
    q = d["q"][(qoff[:-1, None] + i).clamp(max=d["q"].shape[0] - 1)].float()
    k, v = (d[n][(koff[:-1, None] + j).clamp(max=d[n].shape[0] - 1)].float().permute(0, 2, 1, 3).contiguous() for n in "kv")
    q = q.reshape(B, Lq, KV, H // KV, HEAD).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, HEAD)
    x = torch.matmul(q * HEAD ** -0.5, k.transpose(2, 3).contiguous()).reshape(B, H, Lq, Lk)
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    p = (d["lengths"] - d["newLengths"])[:, None] + i  # the queries are the documents' last tokens
    away = p[:, :, None] - j
    if case["slopes"]:
        x = x - d["slopes"][:, None, None] * away.abs()[:, None].float()
    seen = (i[:, None] < d["newLengths"][:, None, None]) & (j < d["lengths"][:, None, None])
    if case["mask"] == "window":
        seen = seen & (away.abs() <= WINDOW // 2)
    elif case["mask"] == "causal":
        seen = seen & (away >= 0)
    elif case["mask"] == "prefix":
        seen = seen & ((away >= 0) | (j < d["prefix"][:, None, None]))
    x = x.masked_fill(~seen[:, None], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    o = torch.matmul(e.reshape(B, KV, -1, Lk), v).reshape(B, H, Lq, HEAD) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return {"o": o.permute(0, 2, 1, 3)[qdoc.long(), qpos.long()].to(t)}


def _plain_weight(d):
    if "w" in d:
        return d["w"].float()
    c = d["codes"]
    if c.dtype == torch.uint8:
        c = torch.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1)
    w = c.float().reshape(c.shape[0], -1, GROUP) * d["scales"].float()[..., None]
    if "zeros" in d:
        w = w + d["zeros"].float()[..., None]
    return w.reshape(c.shape).half().float()  # the format's value: rounded once to 16 bits


def _plain_lora(case, d):
    n, R, N = case["n"], case["R"], case["N"]
    x = d["x"].float()
    y = x @ _plain_weight(d).t()
    if d["bias"] is not None:
        y = y + d["bias"].float()
    # every adapter's inner product, kept where it is the row's own
    s = (x @ d["a"].float().reshape(n * R, -1).t()).reshape(-1, n, R)
    own_rows = d["index"][:, None] == torch.arange(n, device=x.device)
    s = s * (own_rows * d["alpha"])[..., None]
    y = y + s.reshape(-1, n * R) @ d["b"].float().permute(0, 2, 1).reshape(n * R, N)
    return {"y": y.to(TYPES[case["t"]])}


_PLAIN = {"pack": _plain_pack, "rope": _plain_rope, "attn": _plain_attn, "lora": _plain_lora}


# ------------------------------------------------------------------ in 64 bits

def _exact_rope(case, d):
    half = HEAD // 2
    theta = np.empty((case["T"], half), np.float64)
    positions, inv, at = d["positions"].cpu().numpy().astype(np.float64), _frequencies().astype(np.float64), 0
    for axis, pairs in enumerate(_sections(case)):
        for i in range(at, at + pairs):
            theta[:, i] = (positions[axis] * inv[i]).astype(np.float32)
        at += pairs
    z = torch.polar(torch.ones(theta.shape, dtype=torch.float64), torch.from_numpy(theta)).cuda()[:, None, :]
    x = d["qkv"][:, :2 * case["heads"]].double()
    r = torch.complex(x[..., :half], x[..., half:]) * z
    return {"qk": torch.cat([r.real, r.imag], -1)}


def _exact_attn(case, d):
    H, per, out, q0, k0 = case["heads"], case["heads"] // case["kv"], [], 0, 0
    for b, (m, n) in enumerate(zip(d["new"], d["lens"])):
        o = torch.zeros(m, H, HEAD, dtype=torch.float64, device="cuda")
        p, j = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
        seen = torch.ones(m, n, dtype=torch.bool, device="cuda")
        if case["mask"] == "window":
            seen = (p - j).abs() <= WINDOW // 2
        elif case["mask"] != "full":
            seen = j <= p
            if case["mask"] == "prefix":
                seen = seen | (j < int(d["prefix"][b]))
        for h in range(H if m else 0):
            q, k, v = d["q"][q0:q0 + m, h].double(), d["k"][k0:k0 + n, h // per].double(), d["v"][k0:k0 + n, h // per].double()
            x = q @ k.t() / math.sqrt(HEAD)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - float(d["slopes"][h]) * (p - j).abs()
            o[:, h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v
        out.append(o)
        q0, k0 = q0 + m, k0 + n
    return {"o": torch.cat(out)}


def _exact_lora(case, d):
    x = d["x"].double()
    if "w" in d:
        w = d["w"].double()
    else:
        c = d["codes"].cpu().numpy()
        if c.dtype == np.uint8:
            c = np.concatenate([(c & 15)[..., None], (c >> 4)[..., None]], -1).reshape(c.shape[0], -1)
        w = c.astype(np.float64) * np.repeat(d["scales"].cpu().numpy().astype(np.float64), GROUP, 1)
        if "zeros" in d:
            w = w + np.repeat(d["zeros"].cpu().numpy().astype(np.float64), GROUP, 1)
        w = torch.from_numpy(w.astype(np.float16).astype(np.float64)).cuda()
    y = x @ w.t() if d["bias"] is None else torch.addmm(d["bias"].double(), x, w.t())
    for i in range(case["n"]):
        rows = torch.nonzero(d["index"] == i)[:, 0]
        y[rows] += float(d["alpha"][i]) * ((x[rows] @ d["a"][i].double().t()) @ d["b"][i].double().t())
    return {"y": y}


def exact(case, seed):
    """run()'s computed numbers in 64 bits; rows that are only moved have none."""
    if case["op"] == "pack":
        return None
    return {"rope": _exact_rope, "attn": _exact_attn, "lora": _exact_lora}[case["op"]](case, _inputs(case, seed))
