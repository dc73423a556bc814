"""The transformer-block operators of include/ppocr_cuda.h (window attention,
the 8-bit RMS norm, the 4-bit product) against plain 64-bit restatements.

Tolerances are sums of what the arithmetic may lose, taken before the first
run: a rounding to a type loses at most half a step (finfo.eps / 2 of the
value); an f32 sum of n terms at most n * 2^-23 of the sum of magnitudes
(the matrix units truncate, hence 2^-23 and not 2^-24); a 3xTF32 product
2^-20 (each low half is cut to 11 bits, 2^-21 of its operand); 2^x 2^-21.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from ppocr_native_b200 import cuda

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def half_step(t):
    return torch.finfo(DTYPES[t]).eps / 2


# ---------------------------------------------------------------- attention

class Attn:
    """One call's buffers: lanes of `lens` = (queries, keys), self-attention
    rows unless keys differ."""

    def __init__(self, t, lens, heads, kv_heads, d, left=-1, right=-1, sinks=0, seed=0, interleaved=True, room=0,
                 pad=0, scale=None):
        g = torch.Generator("cuda").manual_seed(seed)
        self.t, self.lens, self.heads, self.kv_heads, self.d = t, lens, heads, kv_heads, d
        self.left, self.right, self.sinks = left, right, sinks
        self.scale = d ** -0.5 if scale is None else scale
        dt = DTYPES[t]
        nq = sum(a for a, _ in lens)
        self.own = all(a == b for a, b in lens) and room == 0
        if self.own and interleaved:
            rows = torch.randn(nq + pad, (heads + 2 * kv_heads) * d, generator=g, device="cuda").to(dt)
            self.q, self.k, self.v = (x.unflatten(1, (-1, d)) for x in
                                      rows.split([heads * d, kv_heads * d, kv_heads * d], 1))
            self.begin = [sum(a for a, _ in lens[:i]) for i in range(len(lens))]
        else:
            room = max(room, max([b for _, b in lens] + [1]))
            self.q = torch.randn(max(nq + pad, 1), heads, d, generator=g, device="cuda").to(dt)
            # heads outermost, as a cache may keep them
            self.k, self.v = (torch.randn(kv_heads, len(lens) * room, d, generator=g, device="cuda").to(dt)
                              .transpose(0, 1) for _ in range(2))
            self.begin = [i * room for i in range(len(lens))]
        self.out = torch.full((max(nq + pad, 1), heads, d), 7.0, device="cuda").to(dt)
        self.offsets = torch.tensor([sum(a for a, _ in lens[:i]) for i in range(len(lens) + 1)], device="cuda")
        self.k_begin = torch.tensor(self.begin, device="cuda")
        self.k_len = torch.tensor([b for _, b in lens], dtype=torch.int32, device="cuda")

    def shape(self, **kw):
        return cuda.AttentionShape(**({
            "type": self.t, "lanes": len(self.lens), "heads": self.heads, "kv_heads": self.kv_heads,
            "head_dim": self.d, "q_rows": self.q.shape[0], "kv_rows": self.k.shape[0], "scale": self.scale,
            "left": self.left, "right": self.right, "sinks": self.sinks, "q_strides": self.q.stride()[:2],
            "k_strides": self.k.stride()[:2], "v_strides": self.v.stride()[:2],
            "out_strides": self.out.stride()[:2], "max_q": max([a for a, _ in self.lens] + [0]),
            "max_k": max([b for _, b in self.lens] + [0])} | kw))

    def call(self, shape=None, stream=None, implied=False):
        cuda.attention_window(shape or self.shape(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(),
                              self.out.data_ptr(), self.offsets.data_ptr(),
                              None if implied else self.k_begin.data_ptr(),
                              None if implied else self.k_len.data_ptr(),
                              stream or torch.cuda.current_stream().cuda_stream)

    def check(self):
        share = self.heads // self.kv_heads
        at = 0
        for (nq, nk), begin in zip(self.lens, self.begin):
            q = self.q[at:at + nq].double()
            k, v = (x[begin:begin + nk].double().repeat_interleave(share, 1) for x in (self.k, self.v))
            p, j = torch.arange(nq, device="cuda")[:, None] + nk - nq, torch.arange(nk, device="cuda")[None]
            seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
            if self.right >= 0:
                seen &= j <= p + self.right
            if self.left >= 0:
                seen &= (j >= p - self.left) | (j < self.sinks)
            s = torch.einsum("ihd,jhd->hij", q, k.nan_to_num(0, 0, 0)) * self.scale
            odd_k = ~k.isfinite().all(2).T  # [h, j]: a key that is not finite, wherever seen, spoils the row
            s = s.masked_fill(~seen, -math.inf)
            w = torch.softmax(s, 2).nan_to_num(0)
            odd_v = ~v.isfinite()
            want = torch.einsum("hij,jhd->ihd", w, v.nan_to_num(0, 0, 0))
            spoilt = (seen[None] & odd_k[:, None]).any(2).T[:, :, None] | \
                (torch.einsum("hij,jhd->ihd", seen.double().expand(self.heads, -1, -1), odd_v.double()) > 0)
            got = self.out[at:at + nq].double()
            assert not got[spoilt.expand_as(got)].isfinite().any() if bool(spoilt.any()) else True
            mags = torch.einsum("hij,jhd->ihd", w, v.nan_to_num(0, 0, 0).abs())
            # the scores' error, doubled since numerator and sum both move
            pairs = torch.einsum("ihd,jhd->hij", q.abs(), k.nan_to_num(0, 0, 0).abs()) * abs(self.scale)
            pairs = pairs.masked_fill(~seen, 0).amax(2).T[:, :, None] if nk else torch.zeros(nq, self.heads, 1, device="cuda")
            product = 2.0 ** -20 if self.t == "f32" else 0.0
            ds = pairs * (product + (self.d + 4) * 2.0 ** -23)
            weight = product if self.t == "f32" else half_step(self.t)
            tol = mags * (2 * ds + weight + (nk + 8) * 2.0 ** -23 + 2.0 ** -21)
            tol = tol + half_step(self.t) * (want.abs() + tol) + 1e-30
            if self.t == "f16":
                # weights and outputs below f16's smallest normal number round to steps of 2^-24
                tol = tol + 2.0 ** -25 * (1 + (v.nan_to_num(0, 0, 0).abs().sum(0)[None] if nk else 0))
            ok = spoilt.expand_as(got) | ((got - want).abs() <= tol)
            assert bool(ok.all()), float(((got - want).abs() / tol)[~ok].nan_to_num(math.inf).max())
            at += nq
        rest = self.out[at:].float()
        assert bool((rest == 7.0).all()), "rows in no lane were written"


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (7, 0, 3), (40, 25, 2), (-1, 5, 0), (12, -1, 5), (100, 0, 70), (0, 3, 1)]


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
def test_attention_lines(cuda_mod, t, left, right, sinks):
    # one step, empty lanes, tile borders and odd lengths, 15 as head size
    lens = [(n, n) for n in (1, 0, 5, 63, 64, 65, 200, 17, 0, 129)]
    a = Attn(t, lens, 8, 8, 15, left, right, sinks, seed=1, pad=3)
    a.call()
    a.check()
    first = a.out.clone()
    a.call(implied=True)  # keys named by the queries' own rows: the same call
    assert torch.equal(a.out, first)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [1, 2, 8, 16, 20, 33, 40, 64, 72, 80, 96, 100, 120, 128])
def test_attention_head_sizes(cuda_mod, t, d):
    a = Attn(t, [(150, 150), (70, 70), (257, 257)], 4, 2, d, 60, 10, 4, seed=d, pad=2)
    a.call()
    a.check()
    b = Attn(t, [(1, 300), (1, 1), (1, 90)], 4, 2, d, 100, 0, 4, seed=d, room=310, pad=1)
    b.call()
    b.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 16), (8, 2), (16, 1), (40, 1)])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (511, 0, 4), (30, 0, 100), (0, 0, 0)])
def test_attention_steps(cuda_mod, t, heads, kv_heads, left, right, sinks):
    # one new row behind caches of every kind of length; an empty cache's only key is its own
    lens = [(1, n) for n in (1, 2, 31, 32, 33, 500, 1700, 129)] + [(0, 60), (1, 0)]
    a = Attn(t, lens, heads, kv_heads, 64, left, right, sinks, seed=3, room=1705, pad=2)
    a.call()
    a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (50, 0, 2), (3, 1, 0)])
def test_attention_rows_that_see_nothing(cuda_mod, t, left, right, sinks):
    # more queries than keys: the first ones stand before the first key
    a = Attn(t, [(90, 20), (5, 0), (3, 1), (130, 70), (4, 4)], 4, 4, 32, left, right, sinks, seed=4, room=80, pad=5)
    a.call()
    a.check()
    if right >= 0:
        assert bool((a.out[:90 - 20 - right] == 0).all()) and bool((a.out[90:95] == 0).all())


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("steps", [False, True])
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_masked_places_may_hold_anything(cuda_mod, t, steps, bad, d):
    lens = [(2, 600), (1, 77)] if steps else [(300, 300), (77, 77)]
    a = Attn(t, lens, 4, 2, d, 50, 0, 3, seed=5, interleaved=False, room=650)
    # outside every window, or seen by some queries only
    a.v[100] = bad
    a.v[120, 1, 7] = bad
    a.k[101, 0] = bad
    a.k[630:650] = bad
    a.v[630:650] = bad
    a.k[650 + 77:] = bad
    a.v[650 + 77:] = bad
    a.call()
    a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("steps", [False, True])
def test_attention_large_values_in_masked_places(cuda_mod, t, d, steps):
    # a weight of nearly nothing would show here: hidden keys have none at all
    lens = [(2, 600), (1, 77)] if steps else [(300, 300), (77, 77)]
    a = Attn(t, lens, 16, 16, d, 50, 0, 3, seed=15, interleaved=False, room=650)
    huge = 6e4 if t == "f16" else 3e38
    a.v[100:116] = huge
    a.v[400:420] = -huge
    a.v[630:650] = huge
    a.call()
    a.check()
    # far below the others' scores: a weight of nothing, seen or not
    if not steps:
        b = Attn(t, lens, 16, 16, d, 200, 0, 3, seed=16, interleaved=False, room=300)
        b.q[..., 0], b.k[..., 0] = 16, 0
        b.k[100:140, :, 0] = -16 * d ** 0.5
        b.v[100:140] = huge
        b.call()
        got = b.out[150:300].float()
        assert bool((got.abs() < 8).all())


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_keys_of_no_number(cuda_mod, t, d):
    # at every place of a tile: all the rows that see it, and no other
    for j in (96, 97, 98, 99, 102, 103, 111, 127, 128, 135):
        a = Attn(t, [(300, 300)], 16, 16, d, 50, 0, 3, seed=j, interleaved=False)
        a.k[j, :, d // 2] = math.nan
        a.call()
        a.check()
        assert bool(a.out[j:j + 51].isnan().all()) and bool(a.out[:j].isfinite().all()) and bool(a.out[j + 51:].isfinite().all())


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_attention_lowest_scores(cuda_mod, t):
    # scores at the type's lowest values: no sum of weights may vanish
    a = Attn(t, [(70, 70), (1, 70)], 2, 2, 64, 20, 0, 1, seed=6, interleaved=False, room=70, scale=1.0)
    a.q *= 0
    a.k *= 0
    a.q[..., 0] = 1
    a.k[..., 0] = -6e4 if t == "f16" else -3e38
    a.call()
    a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [40, 128])
@pytest.mark.parametrize("steps", [False, True])
def test_attention_maxima_that_grow(cuda_mod, t, d, steps):
    # keys whose scores rise along the lane, far past the last maximum tile by
    # tile, and fall again: the running sums are rescaled both ways
    lens = [(2, 900), (1, 700)] if steps else [(700, 700), (130, 130)]
    a = Attn(t, lens, 4, 2, d, 400, 30, 5, seed=11, interleaved=False, room=901)
    rise = torch.linspace(0, 6, a.k.shape[0] // 2, device="cuda")
    a.k.mul_(torch.cat([rise, rise.flip(0)])[:, None, None].to(a.k.dtype))
    a.call()
    a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,left,right,sinks", [(128, 700, 0, 4), (64, -1, -1, 0), (80, 300, 300, 130)])
def test_attention_one_long_lane(cuda_mod, t, d, left, right, sinks):
    a = Attn(t, [(2300, 2300)], 4, 2, d, left, right, sinks, seed=12, pad=1)
    a.call()
    a.check()


@gpu
def test_attention_many_lanes_of_steps(cuda_mod):
    # more lanes than are sorted by length, and fewer, empty ones among them
    for lanes in (300, 200):
        lens = [(1, 1 + (i * 37) % 210) if i % 9 else (0, 5) for i in range(lanes)]
        a = Attn("bf16", lens, 8, 2, 64, 100, 0, 2, seed=13, room=211, pad=2)
        a.call()
        a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [16, 40, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (2, 2), (12, 1)])
@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (400, 3, 9), (-1, 0, 0), (290, 0, 40)])
def test_attention_some_queries_over_many_keys(cuda_mod, t, d, heads, kv_heads, left, right, sinks):
    # tiles of 16 rows that hold several queries and heads, the last one short
    lens = [(33, 700), (5, 300), (20, 20), (0, 50), (40, 10), (1, 900), (16, 33)]
    a = Attn(t, lens, heads, kv_heads, d, left, right, sinks, seed=21, room=903, pad=4)
    a.call()
    a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [20, 64, 120])
def test_attention_many_short_lanes(cuda_mod, t, d):
    # heads that share a key head in one tile, keys too few to split
    lens = [(1 + i % 3, 1 + (i * 7) % 60) if i % 11 else (0, 5) for i in range(60)]
    a = Attn(t, lens, 16, 2, d, 40, 0, 3, seed=22, room=61, pad=2)
    a.call()
    a.check()
    # one head a key head, more tiles than SMs
    lens = [(16 - i % 4, 300 + 13 * i) for i in range(20)]
    a = Attn(t, lens, 8, 8, d, 350, 0, 1, seed=23, room=560, pad=1)
    a.call()
    a.check()


@gpu
def test_attention_hints_size_the_launch_only(cuda_mod):
    a = Attn("bf16", [(300, 300), (9, 9), (150, 150)], 4, 2, 64, 64, 0, 2, seed=7)
    for hint in ((1, 1), (0, 0), (10 ** 6, 10 ** 6), (20, 300)):
        a.out.fill_(7.0)
        a.call(a.shape(max_q=hint[0], max_k=hint[1]))
        a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_attention_strides_and_alignment(cuda_mod, t, shift):
    # rows, heads and bases off every vector width
    dt, n, h, d = DTYPES[t], 150, 3, 24
    a = Attn(t, [(n, n)], h, h, d, 30, 6, 2, seed=8)
    def apart(x):
        flat = torch.zeros(n * (h * (d + shift) + shift) + 64, dtype=dt, device="cuda")
        y = flat[shift:].as_strided((n, h, d), (h * (d + shift) + shift, d + shift, 1), shift)
        y.copy_(x)
        return y
    a.q, a.k, a.v, a.out = apart(a.q), apart(a.k), apart(a.v), apart(a.out)
    a.call()
    a.check()
    b = Attn(t, [(1, 90)], 4, 1, 24, 30, 0, 2, seed=8, room=93)
    k = torch.zeros(93 * 40 + 8, dtype=dt, device="cuda")[shift:].as_strided((93, 1, 24), (24 + shift, 24, 1), shift)
    k.copy_(b.k)
    b.k = k
    b.call()
    b.check()


@gpu
def test_attention_offsets_past_32_bits(cuda_mod):
    # a cache of more than 2^32 elements; the lane lies at its end
    rows, h, d = (1 << 32) // (8 * 128) + 500, 8, 128
    big = torch.zeros(rows, h, d, dtype=torch.bfloat16, device="cuda")
    for q_len in (1, 200):
        a = Attn("bf16", [(q_len, 400)], h, h, d, 300, 0, 4, seed=9, room=400)
        big[-450:-50] = a.k
        want_v = a.v
        a.k, a.begin, a.k_begin = big, [rows - 450], torch.tensor([rows - 450], device="cuda")
        a.v = big
        a.call()
        a.check()
        del want_v
    del big
    torch.cuda.empty_cache()


@gpu
def test_attention_lane_arrays_are_cut_to_the_tensors(cuda_mod):
    a = Attn("f16", [(40, 40), (30, 30)], 2, 2, 32, 10, 0, 1, seed=10, interleaved=False, room=40)
    want = a.out
    a.call()
    full, a.out = a.out, torch.full_like(a.out, 7.0)
    # the second lane's rows claim to run far past the tensors
    a.offsets = torch.tensor([0, 40, 10 ** 12], device="cuda")
    a.k_len = torch.tensor([40, 10 ** 9], dtype=torch.int32, device="cuda")
    a.k_begin = torch.tensor([0, 40], device="cuda")
    a.call()
    torch.cuda.synchronize()
    assert torch.equal(a.out[:40], full[:40]) and want is full
    a.offsets = torch.tensor([-5, 10 ** 14, 3], device="cuda")
    a.k_begin = torch.tensor([-(10 ** 15), 10 ** 15], device="cuda")
    a.k_len = torch.tensor([-3, 50], dtype=torch.int32, device="cuda")
    a.call()
    torch.cuda.synchronize()


# ---------------------------------------------------------------- the norm

def norm_check(t, x, r, gamma, eps, group, s, y, scales):
    c = x.shape[1]
    want = x.double() + (r.double() if r is not None else 0)
    u = half_step(t) if t != "f32" else 0.0
    if s is not None:
        least = torch.finfo(DTYPES[t]).smallest_normal * torch.finfo(DTYPES[t]).eps  # below it steps are this wide
        assert bool(((s.double() - want).abs() <= want.abs() * (u + 2.0 ** -23) + least).all())
    n = want / (want.square().mean(1, keepdim=True) + eps).sqrt() * gamma.double()
    width = group or c
    groups = -(-c // width)
    each = torch.arange(c, device="cuda") // width
    peak = torch.zeros(x.shape[0], groups, dtype=torch.float64, device="cuda")
    peak.scatter_reduce_(1, each.expand(x.shape[0], -1), n.abs(), "amax")
    # the sum s, its squares' sum (at most a chain of c), the root, the quotient and the products
    lose = (c / 2 + 16) * 2.0 ** -24
    assert bool(((scales.double() - peak / 448).abs() <= peak / 448 * lose + 2.0 ** -149).all())
    got = y.view(torch.float8_e4m3fn).double() * scales.double()[:, each]
    step = torch.maximum(n.abs() * 2.0 ** -4, peak[:, each] / 448 * 2.0 ** -10)
    assert bool(((got - n).abs() <= step * (1 + 2.0 ** -10) + n.abs() * 2 * lose + 2.0 ** -149 * 448).all())


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("rows,c", [(1, 1), (40, 120), (3, 8), (7, 33), (130, 256), (5, 264), (9, 512), (4, 1111),
                                    (6, 2048), (3, 2056), (5, 4096), (2, 8200), (3, 16384), (2, 20000), (1, 32768)])
def test_norm(cuda_mod, t, group, rows, c):
    g = torch.Generator("cuda").manual_seed(c)
    x, r = (torch.randn(rows, c, generator=g, device="cuda").to(DTYPES[t]) for _ in range(2))
    gamma = torch.randn(c, generator=g, device="cuda")
    groups = -(-c // group) if group else 1
    for residual, keep in ((r, True), (r, False), (None, False), (None, True)):
        s, y = torch.empty_like(x), torch.empty(rows, c, dtype=torch.uint8, device="cuda")
        scales = torch.empty(rows, groups, device="cuda")
        cuda.rms_norm_e4m3(cuda.RmsNormShape(t, rows, c, group, 1e-5), x.data_ptr(),
                           residual.data_ptr() if residual is not None else None, gamma.data_ptr(),
                           s.data_ptr() if keep else None, y.data_ptr(), scales.data_ptr(),
                           torch.cuda.current_stream().cuda_stream)
        norm_check(t, x, residual, gamma, 1e-5, group, s if keep else None, y, scales)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("rows,c", [(9001, 100), (4001, 500), (2600, 1001), (2600, 1024), (1300, 2047), (1301, 4096), (700, 5003),
                                    (700, 8192)])
def test_norm_more_rows_than_blocks(cuda_mod, t, group, rows, c):
    g = torch.Generator("cuda").manual_seed(c)
    x, r = (torch.randn(rows, c, generator=g, device="cuda").to(DTYPES[t]) for _ in range(2))
    gamma = torch.randn(c, generator=g, device="cuda")
    s, y = torch.empty_like(x), torch.empty(rows, c, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, -(-c // group) if group else 1, device="cuda")
    cuda.rms_norm_e4m3(cuda.RmsNormShape(t, rows, c, group, 1e-5), x.data_ptr(), r.data_ptr(), gamma.data_ptr(),
                       s.data_ptr(), y.data_ptr(), scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
    norm_check(t, x, r, gamma, 1e-5, group, s, y, scales)


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c,row", [(120, 121), (264, 272), (100, 104), (1000, 1003)])
def test_norm_strides_and_in_place(cuda_mod, t, c, row):
    rows = 37
    x, r = (torch.randn(rows, row, device="cuda").to(DTYPES[t]) for _ in range(2))
    gamma = torch.rand(c, device="cuda")
    x0, r0 = x.clone(), r.clone()
    y = torch.full((rows, row), 9, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, 1, device="cuda")
    shape = cuda.RmsNormShape(t, rows, c, 0, 1e-6, row, row, row, row)
    cuda.rms_norm_e4m3(shape, x.data_ptr(), r.data_ptr(), gamma.data_ptr(), r.data_ptr(), y.data_ptr(),
                       scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
    norm_check(t, x0[:, :c], r0[:, :c], gamma, 1e-6, 0, r[:, :c], y[:, :c].contiguous(), scales)
    assert torch.equal(r[:, c:], r0[:, c:]) and bool((y[:, c:] == 9).all()) and torch.equal(x, x0)
    want, r = r.clone(), r0.clone()
    cuda.rms_norm_e4m3(shape, x.data_ptr(), r.data_ptr(), gamma.data_ptr(), x.data_ptr(), y.data_ptr(),
                       scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert torch.equal(x[:, :c], want[:, :c]) and torch.equal(r, r0)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("group", [0, 32])
def test_norm_rows_of_zeros_and_of_no_numbers(cuda_mod, t, group):
    rows, c = 6, 160
    x = torch.randn(rows, c, device="cuda").to(DTYPES[t])
    x[0] = 0
    x[1, 5] = math.nan
    x[2, 5] = math.inf
    x[3, 32:64] = 0
    y, groups = torch.empty(rows, c, dtype=torch.uint8, device="cuda"), 5 if group else 1
    scales, gamma = torch.empty(rows, groups, device="cuda"), torch.ones(c, device="cuda")
    cuda.rms_norm_e4m3(cuda.RmsNormShape(t, rows, c, group, 0.0), x.data_ptr(), None, gamma.data_ptr(), None,
                       y.data_ptr(), scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
    f = y.view(torch.float8_e4m3fn).float()
    # with eps 0 a row of zeros is 0 / 0: not a number, as the formula says
    assert bool(scales[0].isnan().all()) and bool(f[0].isnan().all())
    assert bool(scales[1].isnan().all()) and bool(f[1].isnan().all())
    assert bool(scales[2, 0].isnan()) and bool(f[2, :32].isnan().all())
    if group:
        assert float(scales[3, 1]) == 0 and bool((f[3, 32:64] == 0).all())
    for i in (4, 5):
        norm_check(t, x[i:i + 1], None, gamma, 0.0, group, None, y[i:i + 1], scales[i:i + 1])
    cuda.rms_norm_e4m3(cuda.RmsNormShape(t, rows, c, group, 1e-6), x.data_ptr(), None, gamma.data_ptr(), None,
                       y.data_ptr(), scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert bool((scales[0] == 0).all()) and bool((y[0] == 0).all())


# ---------------------------------------------------------------- the 4-bit product

class Q4:
    def __init__(self, xt, yt, m, k, n, group, zeros=True, bias=True, scale_type="f16", w_pad=0, shift=0, x_group=0,
                 seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.args = xt, yt, scale_type, m, k, n, group, x_group
        groups, half = -(-k // group), (k + 1) // 2
        self.x = torch.randn(m, k, generator=g, device="cuda")
        self.x_scales = None
        if xt == "e4m3":
            width = group if x_group else k
            self.x_scales = torch.rand(m, groups if x_group else 1, generator=g, device="cuda") + 0.5
            self.x = (self.x * 50).clamp(-448, 448).to(torch.float8_e4m3fn)
            self.value = self.x.double() * self.x_scales.double()[:, torch.arange(k, device="cuda") // width]
        else:
            self.x = self.x.to(DTYPES[xt])
            self.value = self.x.double()
        flat = torch.randint(0, 256, (n * (half + w_pad) + shift + 16,), generator=g, device="cuda", dtype=torch.uint8)
        self.w = flat[shift:].as_strided((n, half), (half + w_pad, 1), shift)
        self.scales = torch.randn(n, groups, generator=g, device="cuda").to(DTYPES[scale_type])
        self.zeros = torch.randint(0, 16, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
        self.bias = torch.randn(n, generator=g, device="cuda") if bias else None
        self.y = torch.empty(m, n, dtype=DTYPES[yt], device="cuda")

    def call(self, **kw):
        xt, yt, st, m, k, n, group, x_group = self.args
        p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
        cuda.matvec_q4(cuda.MatvecQ4Shape(xt, yt, st, m, k, n, group, x_group, w_row=self.w.stride(0), **kw), p(self.x),
                       p(self.x_scales), p(self.w), p(self.scales), p(self.zeros), p(self.bias), p(self.y),
                       torch.cuda.current_stream().cuda_stream)

    def check(self):
        _, yt, _, m, k, n, group, _ = self.args
        q = torch.stack([self.w & 15, self.w >> 4], 2).flatten(1)[:, :k].double()
        each = torch.arange(k, device="cuda") // group
        w = (q - (self.zeros.double()[:, each] if self.zeros is not None else 8)) * self.scales.double()[:, each]
        want, mags = self.value @ w.T, self.value.abs() @ w.T.abs()
        if self.bias is not None:
            want, mags = want + self.bias.double(), mags + self.bias.double().abs()
        tol = mags * (k + 16) * 2.0 ** -23 + half_step(yt) * want.abs() + (2.0 ** -25 if yt == "f16" else 0)
        over = want.abs() > 65504 if yt == "f16" else torch.zeros_like(want, dtype=torch.bool)
        ok = over | ((self.y.double() - want).abs() <= tol)
        assert bool(ok.all()), float(((self.y.double() - want).abs() / tol)[~ok].max())


@gpu
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,k,n,group", [(1, 1, 1, 32), (1, 120, 360, 32), (2, 64, 17, 64), (3, 1000, 777, 32),
                                         (5, 257, 100, 128), (8, 4096, 64, 128), (9, 640, 130, 64), (16, 1024, 48, 128),
                                         (17, 333, 50, 96), (32, 2049, 40, 32), (1, 8192, 300, 128), (1, 40000, 33, 256),
                                         (31, 5000, 20, 64), (1, 100, 40000, 32), (16, 4096, 20000, 64),
                                         (2, 2048, 9000, 32), (20, 20000, 70, 128), (9, 70000, 40, 64), (2, 70000, 20, 128)])
def test_q4(cuda_mod, xt, zeros, m, k, n, group):
    for yt in ("f32", "bf16", "f16"):
        # rows on 16 bytes and rows side by side
        half = (k + 1) // 2
        for pad, st in ((-half % 16, "f16"), (0, "f32" if yt == "f32" else "bf16")):
            a = Q4(xt, yt, m, k, n, group, zeros, bias=pad > 0, scale_type=st, w_pad=pad, seed=m + k)
            a.call()
            a.check()


@gpu
@pytest.mark.parametrize("m,k,n,group", [(1, 120, 50, 32), (7, 1000, 90, 128), (16, 4096, 64, 64), (32, 640, 33, 96)])
def test_q4_group_scales_of_x_and_odd_places(cuda_mod, m, k, n, group):
    a = Q4("e4m3", "f32", m, k, n, group, x_group=group, seed=1)
    a.call()
    a.check()
    for xt in ("f32", "f16", "bf16", "e4m3"):
        a = Q4(xt, "bf16", m, k, n, group, w_pad=3, shift=1, seed=2)
        x = torch.zeros(m, k + 3, dtype=a.x.dtype, device="cuda")
        y = torch.zeros(m, n + 5, dtype=a.y.dtype, device="cuda")
        x[:, :k].copy_(a.x)
        a.x, a.y = x, y
        a.call(x_row=k + 3, y_row=n + 5)
        assert bool((y[:, n:] == 0).all())
        a.y = y[:, :n]
        a.check()


@gpu
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
def test_q4_rows_of_x_are_apart(cuda_mod, xt):
    # a row with an infinity or a NaN spoils itself alone; the largest f32 stays exact
    a = Q4(xt, "f32", 4, 300, 40, 32, zeros=False, bias=False, seed=3)
    a.call()
    clean = a.y.clone()
    a.x[1, 7] = math.nan
    a.x[2, 299] = math.inf
    a.call()
    assert torch.equal(a.y[[0, 3]], clean[[0, 3]])
    assert bool(a.y[1].isnan().all()) and not bool(a.y[2].isfinite().any())
    if xt == "f32":
        a.x.fill_(0.0)
        a.x[0, 5] = torch.finfo(torch.float32).max
        a.scales.fill_(2.0 ** -5)
        a.value = a.x.double()
        a.call()
        a.check()


@gpu
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("m,k,n,group", [(1, 700, 90, 32), (2, 700, 90, 64), (2, 5000, 40, 128), (1, 33, 17, 32)])
def test_q4_one_and_two_rows_with_no_numbers(cuda_mod, xt, m, k, n, group):
    # whole-number sums have no infinity: such a row is done another way, the
    # row beside it as before
    a = Q4(xt, "f32", m, k, n, group, seed=4)
    a.call()
    a.check()
    clean = a.y.clone()
    x = a.x.float()
    x[0, k // 2] = math.nan
    a.x = x.to(a.x.dtype)
    a.call()
    assert bool(a.y[0].isnan().all()) and torch.equal(a.y[1:], clean[1:])
    if xt != "e4m3":
        x[0, k // 2] = -math.inf
        a.x = x.to(a.x.dtype)
        a.call()
        assert not bool(a.y[0].isfinite().any()) and torch.equal(a.y[1:], clean[1:])
        # magnitudes far apart: the largest decides the step, 2^-31 of it
        tiny = torch.finfo(torch.float32).tiny if xt != "f16" else 2.0 ** -14
        x = a.value.float() * tiny
        a.x = x.to(a.x.dtype)
        a.value = a.x.double()
        a.bias.zero_()
        a.scales.fill_(1.0)
        a.call()
        q = torch.stack([a.w & 15, a.w >> 4], 2).flatten(1)[:, :k].double()
        w = q - a.zeros.double()[:, torch.arange(k, device="cuda") // group]
        off = (a.y.double() - a.value @ w.T).abs()
        assert bool((off <= (a.value.abs() @ w.T.abs()) * (k + 16) * 2.0 ** -23 + 2.0 ** -149 * k).all())


@gpu
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("m,group,zeros", [(1, 128, False), (2, 128, True), (2, 64, True), (1, 32, True)])
def test_q4_large_products_of_one_and_two_rows(cuda_mod, xt, m, group, zeros):
    # odd sizes beyond 2^25 weights
    a = Q4(xt, "f32", m, 4129, 8203, group, zeros=zeros, seed=9)
    a.call()
    a.check()
    clean = a.y.clone()
    x = a.x.float()
    x[0, 2001] = math.nan
    a.x = x.to(a.x.dtype)
    a.call()
    assert bool(a.y[0].isnan().all()) and torch.equal(a.y[1:], clean[1:])


@gpu
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("m,k,n,group", [(3, 9000, 2500, 64), (9, 4200, 2400, 32), (20, 5003, 1200, 128), (32, 8192, 4100, 96)])
def test_q4_many_tiles_of_long_rows(cuda_mod, xt, m, k, n, group):
    # more tiles than SMs and more k than a block's warps hold at once
    a = Q4(xt, "f32", m, k, n, group, seed=17)
    a.call()
    a.check()


@gpu
def test_first_calls_inside_a_capture(cuda_mod, tmp_path):
    # a fresh process whose first call of each operator is a captured one
    import subprocess
    import sys
    from pathlib import Path

    here = Path(__file__).resolve().parent
    code = (f"import sys; sys.path.insert(0, {str(here)!r})\n"
            "import conftest, torch\n"
            "from test_block_ops import block_buffers, block_step\n"
            "dev = block_buffers(20); x = torch.randn(20, 128, device='cuda').half(); start = dev['res'].clone()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    block_step(dev, x, 20)\n"
            "g.replay(); torch.cuda.synchronize(); got = dev['res'].clone(); dev['res'].copy_(start)\n"
            "block_step(dev, x, 20); torch.cuda.synchronize()\n"
            "assert torch.equal(got, dev['res']) and bool(got.isfinite().all())\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@gpu
def test_buffers_elsewhere_are_refused(cuda_mod):
    # plain host memory would fault on the device: refused before any launch
    host = torch.zeros(4096, dtype=torch.float32)
    buffers = [torch.zeros(4096, dtype=torch.float32, device="cuda") for _ in range(9)]
    dev = [b.data_ptr() for b in buffers]
    calls = {
        "attention": lambda p: cuda.attention_window(cuda.AttentionShape("f32", 1, 1, 1, 8, 4, 4, 1.0), *p[:7]),
        "norm": lambda p: cuda.rms_norm_e4m3(cuda.RmsNormShape("f32", 4, 8), *p[:6]),
        "q4": lambda p: cuda.matvec_q4(cuda.MatvecQ4Shape("f32", "f32", "f32", 2, 32, 4, 32), p[0], None, *p[1:6]),
    }
    for name, call in calls.items():
        for i in range(7 if name == "attention" else 6):
            p = list(dev)
            p[i] = host.data_ptr()
            with pytest.raises(cuda.PpocrError) as e:
                call(p)
            assert e.value.code == cuda.E_ARG and "device memory" in str(e.value), (name, i, str(e.value))


# ---------------------------------------------------------------- together

def block_step(dev, x, rows):
    """norm -> 4-bit qkv -> window attention -> 4-bit output layer -> norm, on
    the current stream; the buffers lie in `dev`."""
    s = torch.cuda.current_stream().cuda_stream
    c, h, d = 128, 4, 32
    cuda.rms_norm_e4m3(dev["norm"], x.data_ptr(), dev["res"].data_ptr(), dev["gamma"].data_ptr(), dev["res"].data_ptr(),
                       dev["x8"].data_ptr(), dev["xs"].data_ptr(), s)
    cuda.matvec_q4(dev["qkv_shape"], dev["x8"].data_ptr(), dev["xs"].data_ptr(), dev["wqkv"].data_ptr(),
                   dev["sqkv"].data_ptr(), None, None, dev["qkv"].data_ptr(), s)
    q = dev["qkv"]
    cuda.attention_window(dev["attn"], q.data_ptr(), q.data_ptr() + 2 * h * d, q.data_ptr() + 4 * h * d,
                          dev["att"].data_ptr(), dev["offsets"].data_ptr(), None, None, s)
    cuda.matvec_q4(dev["out_shape"], dev["att"].data_ptr(), None, dev["wo"].data_ptr(), dev["so"].data_ptr(), None, None,
                   dev["y"].data_ptr(), s)
    cuda.rms_norm_e4m3(dev["norm"], dev["y"].data_ptr(), dev["res"].data_ptr(), dev["gamma"].data_ptr(),
                       dev["res"].data_ptr(), dev["x8"].data_ptr(), dev["xs"].data_ptr(), s)


def block_buffers(rows, seed=0):
    c, h, d = 128, 4, 32
    g = torch.Generator("cuda").manual_seed(seed)
    half = dict(dtype=torch.float16, device="cuda")
    dev = {"res": torch.randn(rows, c, generator=g, device="cuda").half(), "gamma": torch.ones(c, device="cuda"),
           "x8": torch.empty(rows, c, dtype=torch.uint8, device="cuda"), "xs": torch.empty(rows, 1, device="cuda"),
           "qkv": torch.empty(rows, 3 * h * d, **half), "att": torch.empty(rows, h, d, **half), "y": torch.empty(rows, c, **half),
           "wqkv": torch.randint(0, 256, (3 * h * d, c // 2), generator=g, device="cuda", dtype=torch.uint8),
           "wo": torch.randint(0, 256, (c, c // 2), generator=g, device="cuda", dtype=torch.uint8),
           "sqkv": torch.full((3 * h * d, 2), 0.02, **half), "so": torch.full((c, 2), 0.02, **half),
           "offsets": torch.tensor([0, 1, rows // 2, rows], device="cuda"),
           "norm": cuda.RmsNormShape("f16", rows, c),
           "qkv_shape": cuda.MatvecQ4Shape("e4m3", "f16", "f16", rows, c, 3 * h * d, 64),
           "out_shape": cuda.MatvecQ4Shape("f16", "f16", "f16", rows, c, c, 64),
           "attn": cuda.AttentionShape("f16", 3, h, h, d, rows, rows, d ** -0.5, 8, 0, 2,
                                       *[(3 * h * d, d)] * 3, (h * d, d), max_q=rows, max_k=rows)}
    return dev


def block_plain(dev, x, res):
    """The same in 64 bits, taking each 8-bit and f16 rounding where the operators put it."""
    c, h, d = 128, 4, 32

    def norm(a, r):
        s = a.double() + r.double()
        n = s / (s.square().mean(1, keepdim=True) + 1e-6).sqrt()
        sc = n.abs().amax(1, keepdim=True) / 448
        return s.half(), (n / sc).float().to(torch.float8_e4m3fn).double() * sc

    def mat(a, w, sc):
        q = torch.stack([w & 15, w >> 4], 2).flatten(1).double() - 8
        return (a @ (q * sc.double().repeat_interleave(64, 1)).T).half()

    res, n = norm(x, res)
    qkv = mat(n, dev["wqkv"], dev["sqkv"]).double()
    q, k, v = (y.unflatten(1, (h, d)) for y in qkv.split(h * d, 1))
    att = torch.zeros_like(q)
    o = dev["offsets"].tolist()
    for a, b in zip(o, o[1:]):
        i, j = torch.arange(b - a, device="cuda")[:, None], torch.arange(b - a, device="cuda")[None]
        seen = (j <= i) & ((j >= i - 8) | (j < 2))
        s = (torch.einsum("ihd,jhd->hij", q[a:b], k[a:b]) * d ** -0.5).masked_fill(~seen, -math.inf)
        att[a:b] = torch.einsum("hij,jhd->ihd", torch.softmax(s, 2), v[a:b])
    y = mat(att.half().double().flatten(1), dev["wo"], dev["so"])
    return norm(y, res)


@gpu
@pytest.mark.parametrize("rows", [3, 20, 32])
def test_block_step(cuda_mod, rows):
    dev = block_buffers(rows)
    x, res = torch.randn(rows, 128, device="cuda").half(), dev["res"].clone()
    block_step(dev, x, rows)
    s, n = block_plain(dev, x, res)
    # five roundings to f16 and one to 8 bits (whose flips at a border move a
    # product's term by a step, 2^-3 of it) through two sums of 128 terms with
    # weights up to 0.16: of the order of 128^0.5 * 0.16 * 2^-8 in the stream
    assert float((dev["res"].double() - s.double()).abs().max()) <= 0.05 * float(s.double().abs().max())
    got = dev["x8"].view(torch.float8_e4m3fn).double() * dev["xs"].double()
    assert float((got - n).norm() / n.norm()) <= 2.0 ** -4


@gpu
def test_block_step_in_a_graph_and_on_two_streams(cuda_mod):
    rows = 20
    devs = [block_buffers(rows, seed=i) for i in range(2)]
    xs = [torch.randn(rows, 128, device="cuda").half() for _ in devs]
    start = [d["res"].clone() for d in devs]
    want = []
    for d, x, r in zip(devs, xs, start):
        block_step(d, x, rows)
        want.append({k: d[k].clone() for k in ("res", "x8", "xs", "att", "y")})
        d["res"].copy_(r)
    torch.cuda.synchronize()
    # at the same time on two streams
    streams = [torch.cuda.Stream() for _ in devs]
    for _ in range(5):
        for s, d, x in zip(streams, devs, xs):
            with torch.cuda.stream(s):
                block_step(d, x, rows)
        torch.cuda.synchronize()
        for d, w, r in zip(devs, want, start):
            for k in w:
                assert torch.equal(d[k], w[k]), k
            d["res"].copy_(r)
        torch.cuda.synchronize()
    # two graphs, replayed at the same time, then with other lanes and inputs
    graphs = []
    for s, d, x in zip(streams, devs, xs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            block_step(d, x, rows)
        graphs.append(g)
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for d, w, r in zip(devs, want, start):
        for k in w:
            assert torch.equal(d[k], w[k]), k
        d["res"].copy_(r)
    devs[0]["offsets"].copy_(torch.tensor([0, 9, 9, 20], device="cuda"))
    xs[0].mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    got = {k: devs[0][k].clone() for k in want[0]}
    devs[0]["res"].copy_(start[0])
    block_step(devs[0], xs[0], rows)
    for k in got:
        assert torch.equal(got[k], devs[0][k]), k


# ---------------------------------------------------------------- refusals (no GPU)

P = 1 << 20  # an address that no refused call reads


def attn_call(q=P, k=2 * P, v=3 * P, out=4 * P, offsets=P, begin=P, length=P, **kw):
    base = dict(type="f16", lanes=2, heads=4, kv_heads=2, head_dim=64, q_rows=10, kv_rows=10, scale=0.1)
    cuda.attention_window(cuda.AttentionShape(**(base | kw)), q, k, v, out, offsets, begin, length)


@pytest.mark.parametrize("code,kw", [
    (cuda.E_ARG, dict(type="e4m3")), (cuda.E_ARG, dict(heads=5)), (cuda.E_ARG, dict(kv_heads=0)), (cuda.E_ARG, dict(heads=0)),
    (cuda.E_ARG, dict(left=-2)), (cuda.E_ARG, dict(right=-2)), (cuda.E_ARG, dict(scale=math.nan)),
    (cuda.E_SIZE, dict(head_dim=0)), (cuda.E_SIZE, dict(head_dim=129)), (cuda.E_SIZE, dict(lanes=65536)),
    (cuda.E_SIZE, dict(heads=1 << 17, kv_heads=1)), (cuda.E_SIZE, dict(q_rows=(1 << 30) + 1)),
    (cuda.E_SIZE, dict(kv_rows=(1 << 30) + 1)), (cuda.E_SIZE, dict(k_strides=((1 << 40) + 1, 64))),
    (cuda.E_SIZE, dict(k_strides=(1 << 40, 64), kv_rows=1 << 20)),
    (cuda.E_ARG, dict(q=0)), (cuda.E_ARG, dict(k=0)), (cuda.E_ARG, dict(v=0)), (cuda.E_ARG, dict(out=0)),
    (cuda.E_ARG, dict(offsets=0)), (cuda.E_ARG, dict(begin=0)), (cuda.E_ARG, dict(length=0)),
    (cuda.E_ARG, dict(q=P + 1)), (cuda.E_ARG, dict(out=P + 1)), (cuda.E_ARG, dict(offsets=P + 4)),
    (cuda.E_ARG, dict(begin=P + 4)), (cuda.E_ARG, dict(length=P + 2)), (cuda.E_ARG, dict(out_strides=(255, 64))),
    (cuda.E_ARG, dict(out_strides=(256, 63))), (cuda.E_ARG, dict(out=P + 128)), (cuda.E_ARG, dict(out=2 * P + 2)),
    (cuda.E_ARG, dict(out=3 * P + 2))])
def test_attention_refuses(code, kw):
    with pytest.raises(cuda.PpocrError) as e:
        attn_call(**kw)
    assert e.value.code == code, str(e.value)
    assert "ppocr_attention_window" in str(e.value)


def norm_call(x=P, residual=2 * P, gamma=3 * P, sum=4 * P, y=5 * P, scales=6 * P, **kw):
    base = dict(type="f16", rows=10, channels=100)
    cuda.rms_norm_e4m3(cuda.RmsNormShape(**(base | kw)), x, residual, gamma, sum, y, scales)


@pytest.mark.parametrize("code,kw", [
    (cuda.E_ARG, dict(type="e4m3")), (cuda.E_ARG, dict(group=16)), (cuda.E_ARG, dict(group=256)), (cuda.E_ARG, dict(eps=-1.0)),
    (cuda.E_ARG, dict(eps=math.nan)), (cuda.E_ARG, dict(eps=math.inf)), (cuda.E_SIZE, dict(channels=0)),
    (cuda.E_SIZE, dict(channels=32769)), (cuda.E_SIZE, dict(rows=(1 << 32) + 1)), (cuda.E_SIZE, dict(x_row=(1 << 32) + 1)),
    (cuda.E_ARG, dict(x=0)), (cuda.E_ARG, dict(gamma=0)), (cuda.E_ARG, dict(y=0)), (cuda.E_ARG, dict(scales=0)),
    (cuda.E_ARG, dict(x=P + 1)), (cuda.E_ARG, dict(residual=P + 1)), (cuda.E_ARG, dict(sum=P + 1)), (cuda.E_ARG, dict(gamma=P + 2)),
    (cuda.E_ARG, dict(scales=P + 2)), (cuda.E_ARG, dict(sum_row=99)), (cuda.E_ARG, dict(y_row=99)),
    (cuda.E_ARG, dict(sum=P + 2)), (cuda.E_ARG, dict(sum=P, sum_row=200)), (cuda.E_ARG, dict(sum=2 * P + 4)),
    (cuda.E_ARG, dict(y=P)), (cuda.E_ARG, dict(y=2 * P)), (cuda.E_ARG, dict(y=4 * P)), (cuda.E_ARG, dict(scales=P)),
    (cuda.E_ARG, dict(scales=5 * P))])
def test_norm_refuses(code, kw):
    with pytest.raises(cuda.PpocrError) as e:
        norm_call(**kw)
    assert e.value.code == code, str(e.value)
    assert "ppocr_rms_norm_e4m3" in str(e.value)


def q4_call(x=P, x_scales=None, w=2 * P, scales=3 * P, zeros=4 * P, bias=5 * P, y=6 * P, **kw):
    base = dict(x_type="f16", y_type="f16", scale_type="f16", rows=4, k=100, n=50, group=32)
    cuda.matvec_q4(cuda.MatvecQ4Shape(**(base | kw)), x, x_scales, w, scales, zeros, bias, y)


@pytest.mark.parametrize("code,kw", [
    (cuda.E_ARG, dict(y_type="e4m3")), (cuda.E_ARG, dict(scale_type="e4m3")), (cuda.E_ARG, dict(group=0)),
    (cuda.E_ARG, dict(group=40)), (cuda.E_ARG, dict(group=1 << 21)), (cuda.E_SIZE, dict(rows=33)), (cuda.E_SIZE, dict(k=0)),
    (cuda.E_SIZE, dict(k=(1 << 20) + 1)), (cuda.E_SIZE, dict(n=(1 << 24) + 1)), (cuda.E_SIZE, dict(w_row=(1 << 32) + 1)),
    (cuda.E_ARG, dict(x=0)), (cuda.E_ARG, dict(w=0)), (cuda.E_ARG, dict(scales=0)), (cuda.E_ARG, dict(y=0)),
    (cuda.E_ARG, dict(x_type="e4m3")), (cuda.E_ARG, dict(x_scales=P)), (cuda.E_ARG, dict(x_type="e4m3", x_scales=7 * P, x_group=64)),
    (cuda.E_ARG, dict(x=P + 1)), (cuda.E_ARG, dict(y=P + 1)), (cuda.E_ARG, dict(scales=P + 1)), (cuda.E_ARG, dict(bias=P + 2)),
    (cuda.E_ARG, dict(w_row=49)), (cuda.E_ARG, dict(y_row=49)), (cuda.E_ARG, dict(y=P)), (cuda.E_ARG, dict(y=2 * P)),
    (cuda.E_ARG, dict(y=3 * P)), (cuda.E_ARG, dict(y=4 * P)), (cuda.E_ARG, dict(y=5 * P))])
def test_q4_refuses(code, kw):
    with pytest.raises(cuda.PpocrError) as e:
        q4_call(**kw)
    assert e.value.code == code, str(e.value)
    assert "ppocr_matvec_q4" in str(e.value)


def test_copied_shapes_stand_alone():
    import copy
    import pickle

    a = cuda.AttentionShape(type="f32", lanes=1, heads=2, kv_heads=2, head_dim=8, q_rows=3, kv_rows=3, scale=1.0)
    for b in (copy.copy(a), copy.deepcopy(a), pickle.loads(pickle.dumps(a))):
        assert b.ref == ctypes.addressof(b) != a.ref and bytes(b) == bytes(a)
        b.lanes = 7
        assert a.lanes == 1 and cuda.AttentionShape.from_address(b.ref).lanes == 7


def test_empty_calls_do_nothing():
    attn_call(lanes=0)
    attn_call(q_rows=0, q=0, out=0)
    norm_call(rows=0, x=0, y=0)
    q4_call(rows=0, x=0)
    q4_call(n=0, w=0)


def test_null_shapes_and_unknown_types():
    lib = cuda.lib()
    assert lib.ppocr_attention_window(None, P, P, P, P, P, None, None, None) == cuda.E_ARG
    assert lib.ppocr_rms_norm_e4m3(None, P, P, P, P, P, P, None) == cuda.E_ARG
    assert lib.ppocr_matvec_q4(None, P, P, P, P, P, P, P, None) == cuda.E_ARG
    with pytest.raises(ValueError):
        cuda.RmsNormShape("int8", 1, 1)
    assert ctypes.sizeof(cuda.AttentionShape) == 128 and ctypes.sizeof(cuda.RmsNormShape) == 56
    assert ctypes.sizeof(cuda.MatvecQ4Shape) == 56
