"""The transformer-block operators' workloads: attention with a sliding window
and sinks, the root-mean-square norm with 8-bit output, and the product with
4-bit weights. Each case names one operator, its sizes and its types; `run`
makes one pass through it, by the framework's kernels (`own`) or in plain
torch operations.
"""

from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def _cuda():
    """The framework's binding (its directory has a hyphen, so it is loaded by path)."""
    name = "ppocr_native_b200"
    if name not in sys.modules:
        root = Path(__file__).resolve().parent.parent / "ppocr-native_b200"
        spec = importlib.util.spec_from_file_location(name, root / "__init__.py", submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name].cuda


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # A page's 44 lines (80 to 1600 pixels wide, 8 pixels a time step) through
        # the recogniser's attention: 8 heads of 15 in f32, q, k, v side by side.
        {"name": "attn page lines f32", "op": "attn", "type": "f32", "lanes": 44, "heads": 8, "kv_heads": 8, "head_dim": 15,
         "q_min": 10, "q_max": 200, "past_min": 0, "past_max": 0, "left": 24, "right": 24, "sinks": 1, "lens": 1},
        # One line read step by step: one query over a short cache, where latency counts.
        {"name": "attn one step bf16", "op": "attn", "type": "bf16", "lanes": 1, "heads": 16, "kv_heads": 4, "head_dim": 64,
         "q_min": 1, "q_max": 1, "past_min": 2000, "past_max": 2000, "left": 511, "right": 0, "sinks": 4, "lens": 2},
        # A server's step: 64 readers at once, long caches of many lengths, grouped key heads.
        {"name": "attn steps bf16", "op": "attn", "type": "bf16", "lanes": 64, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "q_min": 1, "q_max": 1, "past_min": 300, "past_max": 12000, "left": 4095, "right": 0, "sinks": 4, "lens": 3},
        # A whole text read as one long line, causal: the matrix-bound end.
        {"name": "attn long bf16", "op": "attn", "type": "bf16", "lanes": 1, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "q_min": 8192, "q_max": 8192, "past_min": 0, "past_max": 0, "left": 1023, "right": 0, "sinks": 4, "lens": 4},
        # Ragged lines, both neighbours, a head size that is no power of two.
        {"name": "attn ragged f16", "op": "attn", "type": "f16", "lanes": 12, "heads": 8, "kv_heads": 8, "head_dim": 40,
         "q_min": 1, "q_max": 1500, "past_min": 0, "past_max": 0, "left": 128, "right": 128, "sinks": 2, "lens": 5},
        # One line's time steps at the recogniser's width: the smallest norm.
        {"name": "norm one line f32", "op": "norm", "type": "f32", "rows": 40, "channels": 120, "group": 0},
        # A batch of long texts at a wide model: the bandwidth-bound end.
        {"name": "norm wide bf16", "op": "norm", "type": "bf16", "rows": 16384, "channels": 4096, "group": 128},
        # Odd sizes: rows that no vector width divides.
        {"name": "norm odd f16", "op": "norm", "type": "f16", "rows": 1009, "channels": 1111, "group": 0},
        # The recogniser's qkv layer for one time step.
        {"name": "q4 one step f32", "op": "q4", "x": "f32", "y": "f32", "rows": 1, "k": 120, "n": 360, "group": 32, "zeros": False},
        # The class head for sixteen time steps, over the dictionary's 18 710 classes.
        {"name": "q4 head f16", "op": "q4", "x": "f16", "y": "f32", "rows": 16, "k": 120, "n": 18710, "group": 32, "zeros": True},
        # A wide feed-forward layer for one step: the bandwidth-bound end.
        {"name": "q4 wide bf16", "op": "q4", "x": "bf16", "y": "bf16", "rows": 1, "k": 8192, "n": 28672, "group": 128, "zeros": False},
        # A batch of steps behind the norm's 8-bit rows.
        {"name": "q4 steps e4m3", "op": "q4", "x": "e4m3", "y": "bf16", "rows": 16, "k": 4096, "n": 4096, "group": 64, "zeros": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "norm", "q4", "q4"])
    if op == "norm":
        channels = _log(rng, 32, 12288)
        rows = max(1, min(_log(rng, 1, 16384), (16384 * 4096) // channels // 2))
        return {"op": "norm", "type": rng.choice(["f32", "f16", "bf16"]), "rows": rows, "channels": channels,
                "group": rng.choice([0, 32, 64, 128])}
    if op == "q4":
        x = rng.choice(["f32", "f16", "bf16", "e4m3"])
        return {"op": "q4", "x": x, "y": rng.choice(["f32", "f16", "bf16"]), "rows": _log(rng, 1, 32),
                "k": _log(rng, 64, 8192), "n": _log(rng, 64, 28672), "group": rng.choice([32, 64, 128]),
                "zeros": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8])
    share = rng.choice([1, 1, 2, 4])
    step = rng.random() < 0.5
    case = {"op": "attn", "type": rng.choice(["f32", "f16", "bf16"]), "heads": kv_heads * share, "kv_heads": kv_heads,
            "head_dim": rng.choice([15, 16, 20, 32, 33, 40, 64, 72, 80, 96, 120, 128]), "sinks": rng.choice([0, 1, 4, 16])}
    if step:  # one to four new steps at the end of a cache
        lanes = _log(rng, 1, 64)
        case |= {"lanes": lanes, "q_min": 1, "q_max": rng.choice([1, 1, 1, 2, 4]), "past_min": rng.choice([0, 50, 500]),
                 "past_max": _log(rng, 600, max(1500, min(8000, 100000 // lanes))), "left": rng.choice([-1, _log(rng, 16, 4096)]), "right": 0}
    else:  # whole lines, or one long text
        lanes = _log(rng, 1, 64)
        top = max(16, min(4096 if case["heads"] <= 8 else 2048, 12000 // lanes))
        case |= {"lanes": lanes, "q_min": 1 if lanes > 1 else top // 2, "q_max": top, "past_min": 0,
                 "past_max": 0, "left": rng.choice([-1, _log(rng, 8, 1024), _log(rng, 8, 1024)]), "right": rng.choice([0, 0, _log(rng, 1, 256)])}
    return case | {"lens": rng.randrange(1 << 30)}


# ---------------------------------------------------------------- the inputs

def _lens(case):
    """The lanes' query and key counts: part of the case, not of the seed."""
    r = random.Random(case["lens"])
    q = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["lanes"])]
    return q, [n + r.randint(case["past_min"], case["past_max"]) for n in q]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        t, rows, c = TYPES[case["type"]], case["rows"], case["channels"]
        s["x"] = normal(rows, c).to(t)
        # the residual stream: a few channels run far above the others
        s["residual"] = (normal(rows, c) * (1 + 20 * (torch.rand(c, generator=g, device="cuda") > 0.99))).to(t)
        s["gamma"] = 1 + 0.1 * normal(c)
        s["sum"] = torch.empty_like(s["x"])
        s["y"] = torch.empty(rows, c, dtype=torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.empty(rows, -(-c // case["group"]) if case["group"] else 1, device="cuda")
        return s
    if case["op"] == "q4":
        m, k, n, groups = case["rows"], case["k"], case["n"], -(-case["k"] // case["group"])
        x = normal(m, k)
        s["x_scales"] = None
        if case["x"] == "e4m3":
            s["x_scales"] = x.abs().amax(1, keepdim=True) / 448
            x = x / s["x_scales"]
        s["x"] = x.to(TYPES[case["x"]])
        # two weights a byte, the lower four bits first; a row is padded to 16 bytes
        s["w"] = torch.randint(0, 256, (n, -(-k // 32) * 16), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(n, groups, generator=g, device="cuda")) * (0.2 * k ** -0.5)).half()
        s["zeros"] = torch.randint(5, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["bias"] = 0.1 * normal(n)
        s["y"] = torch.empty(m, n, dtype=TYPES[case["y"]], device="cuda")
        return s | {"y_type": case["y"], "x_type": case["x"]}
    t, h, kh, d = TYPES[case["type"]], case["heads"], case["kv_heads"], case["head_dim"]
    nq, nk = _lens(case)
    if case["past_max"] == 0:  # whole lanes: q, k and v side by side in each row, as one product leaves them
        rows = normal(sum(nq), (h + 2 * kh) * d).to(t)
        q, k, v = (x.unflatten(1, (-1, d)) for x in rows.split([h * d, kh * d, kh * d], 1))
        begin = [sum(nq[:i]) for i in range(len(nq))]
    else:  # a cache of rows per lane, each lane with room for the longest
        room = max(nk)
        q = normal(sum(nq), h, d).to(t)
        k, v = (torch.empty(len(nk) * room, kh, d, dtype=t, device="cuda").normal_(generator=g) for _ in range(2))
        begin = [i * room for i in range(len(nk))]
    s |= {"q": q, "k": k, "v": v, "out": torch.empty(sum(nq), h, d, dtype=t, device="cuda"), "scale": d ** -0.5,
          "max_q": max(nq), "max_k": max(nk)}
    s["q_offsets"] = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int64, device="cuda")
    s["k_begin"] = torch.tensor(begin, dtype=torch.int64, device="cuda")
    s["k_len"] = torch.tensor(nk, dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return {"attn": _attn, "norm": _norm, "q4": _q4}[s["op"]](s)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _attn(s):
    q, k, v, out = s["q"], s["k"], s["v"], s["out"]
    if own:
        cuda = _cuda()
        shape = s.get("shape")
        if shape is None:  # the layer's sizes, which a program keeps beside its buffers
            shape = s["shape"] = cuda.AttentionShape(
                type=s["type"], lanes=s["lanes"], heads=s["heads"], kv_heads=s["kv_heads"], head_dim=s["head_dim"],
                q_rows=q.shape[0], kv_rows=k.shape[0], q_strides=q.stride()[:2], k_strides=k.stride()[:2],
                v_strides=v.stride()[:2], out_strides=out.stride()[:2], left=s["left"], right=s["right"], sinks=s["sinks"],
                scale=s["scale"], max_q=s["max_q"], max_k=s["max_k"])
        cuda.attention_window(shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), s["q_offsets"].data_ptr(),
                              s["k_begin"].data_ptr(), s["k_len"].data_ptr(), _stream())
        return out
    first, begin, nk = s["q_offsets"][:-1], s["k_begin"], s["k_len"].long()
    nq = s["q_offsets"][1:] - first
    i, j = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    at = (first[:, None] + i).clamp(max=q.shape[0] - 1)                      # [lane, query]
    from_ = begin[:, None] + torch.minimum(j, (nk[:, None] - 1).clamp(min=0))  # [lane, key]
    p = i + (nk - nq)[:, None]
    p, jj = p[:, :, None], j[None, None, :]
    seen = jj < nk[:, None, None]
    if s["right"] >= 0:
        seen = seen & (jj <= p + s["right"])
    if s["left"] >= 0:
        seen = seen & ((jj >= p - s["left"]) | (jj < s["sinks"]))
    kh, share = s["kv_heads"], s["heads"] // s["kv_heads"]
    qp = q[at].float().unflatten(2, (kh, share)).permute(0, 2, 3, 1, 4)        # [lane, kv head, share, query, d]
    kp = k[from_].float().permute(0, 2, 3, 1)[:, :, None]                      # [lane, kv head, 1, d, key]
    vp = v[from_].float().permute(0, 2, 1, 3)[:, :, None]
    score = (qp @ kp).mul_(s["scale"]).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e @ vp) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    there = i < nq[:, None]
    out[at[there]] = o[there].to(out.dtype)
    return out


def _norm(s):
    x, r, gamma, eps, group = s["x"], s["residual"], s["gamma"], 1e-6, s["group"]
    if own:
        cuda = _cuda()
        shape = s.get("shape")
        if shape is None:
            shape = s["shape"] = cuda.RmsNormShape(type=s["type"], rows=s["rows"], channels=s["channels"], group=group, eps=eps)
        cuda.rms_norm_e4m3(shape, x.data_ptr(), r.data_ptr(), gamma.data_ptr(), s["sum"].data_ptr(), s["y"].data_ptr(),
                           s["scales"].data_ptr(), _stream())
        return s["sum"], s["y"], s["scales"]
    t = x.float() + r.float()
    n = t * torch.rsqrt((t * t).mean(1, keepdim=True) + eps) * gamma
    width = group or s["channels"]
    n = torch.nn.functional.pad(n, (0, -n.shape[1] % width)).unflatten(1, (-1, width))
    scales = n.abs().amax(2) / 448
    y = torch.where(scales[..., None] > 0, n / scales[..., None], 0.0).flatten(1)[:, : s["channels"]]
    return t.to(x.dtype), y.to(torch.float8_e4m3fn), scales


def _q4(s):
    x, w, scales, zeros, bias, y = s["x"], s["w"], s["scales"], s["zeros"], s["bias"], s["y"]
    if own:
        cuda = _cuda()
        shape = s.get("shape")
        if shape is None:
            shape = s["shape"] = cuda.MatvecQ4Shape(x_type=s["x_type"], y_type=s["y_type"], scale_type="f16", rows=s["rows"],
                                                    k=s["k"], n=s["n"], group=s["group"], w_row=w.stride(0))
        cuda.matvec_q4(shape, x.data_ptr(), s["x_scales"].data_ptr() if s["x_scales"] is not None else None, w.data_ptr(),
                       scales.data_ptr(), zeros.data_ptr() if zeros is not None else None, bias.data_ptr(), y.data_ptr(), _stream())
        return y
    q = torch.stack([w & 15, w >> 4], 2).flatten(1)[:, : s["k"]].float()
    each = torch.arange(s["k"], device="cuda") // s["group"]
    q = (q - (zeros.float()[:, each] if zeros is not None else 8.0)).mul_(scales.float()[:, each])
    xf = x.float() if s["x_scales"] is None else x.float() * s["x_scales"]
    return (xf @ q.T + bias).to(y.dtype)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["channels"], BYTES[case["type"]]
        scales = case["rows"] * (-(-case["channels"] // case["group"]) if case["group"] else 1)
        return {"bytes": n * (3 * b + 1) + 4 * scales + 4 * case["channels"], "flops": 8 * n}
    if case["op"] == "q4":
        m, k, n = case["rows"], case["k"], case["n"]
        groups = n * -(-k // case["group"])
        return {"bytes": n * -(-k // 2) + groups * (3 if case["zeros"] else 2) + 4 * n + m * k * BYTES[case["x"]]
                + m * n * BYTES[case["y"]], "flops": 2 * m * k * n}
    nq, nk = _lens(case)
    pairs = rows = 0
    left, right, sinks = case["left"], case["right"], case["sinks"]
    for a, b in zip(nq, nk):
        lowest = b  # the first key behind the sinks that any query of the lane sees
        for p in range(b - a, b):
            hi = b if right < 0 else min(b, p + right + 1)
            lo = 0 if left < 0 else min(max(0, p - left), hi)
            pairs += max(0, hi - lo) + min(lo, sinks, hi)
            lowest = min(lowest, lo)
        rows += b - lowest + min(lowest, sinks)
    d, b = case["head_dim"], BYTES[case["type"]]
    return {"bytes": b * d * (2 * sum(nq) * case["heads"] + 2 * rows * case["kv_heads"]), "flops": 4 * d * case["heads"] * pairs}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        t = s["x"].double() + s["residual"].double()
        n = t / torch.sqrt(t.square().sum(1, keepdim=True) / case["channels"] + 1e-6) * s["gamma"].double()
        parts = torch.split(n, case["group"] or case["channels"], 1)
        scales = [part.abs().max(1, keepdim=True).values / 448 for part in parts]
        y = torch.cat([part / sc for part, sc in zip(parts, scales)], 1)
        return t, y, torch.cat(scales, 1)
    if case["op"] == "q4":
        x = s["x"].double()
        if s["x_scales"] is not None:
            x = x * s["x_scales"].double()
        y = s["bias"].double().repeat(case["rows"], 1)
        k, group = case["k"], case["group"]
        low, high = (s["w"] & 15).double(), (s["w"] >> 4).double()
        for g in range(-(-k // group)):  # a group's products, then its scale
            ks = torch.arange(g * group, min(k, (g + 1) * group), device="cuda")
            w = torch.where(ks % 2 == 0, low[:, ks // 2], high[:, ks // 2])
            w = w - (s["zeros"][:, g, None].double() if s["zeros"] is not None else 8)
            y += (x[:, ks] @ w.T) * s["scales"][:, g].double()
        return y
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    nq, nk = _lens(case)
    share, at = case["heads"] // case["kv_heads"], 0
    for b, (a, c) in enumerate(zip(nq, nk)):
        begin = int(s["k_begin"][b])
        p = torch.arange(c - a, c, device="cuda")[:, None]
        j = torch.arange(c, device="cuda")[None, :]
        hidden = torch.zeros(a, c, dtype=torch.bool, device="cuda")
        if case["right"] >= 0:
            hidden |= j > p + case["right"]
        if case["left"] >= 0:
            hidden |= (j < p - case["left"]) & (j >= case["sinks"])
        for h in range(case["heads"]):
            k, v = (s[x][begin:begin + c, h // share].double() for x in ("k", "v"))
            score = (s["q"][at:at + a, h].double() @ k.T) * case["head_dim"] ** -0.5
            score[hidden] = -math.inf
            out[at:at + a, h] = torch.nan_to_num(torch.softmax(score, 1)) @ v
        at += a
    return out
