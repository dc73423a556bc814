"""The transformer-block operators at their edges: values far apart, rows that
are not finite, clusters, lanes longer than their hints, buffers in host
memory. Tolerances as in test_block_ops, unless a test derives its own."""

from __future__ import annotations

import math
from pathlib import Path

import pytest
import torch

from ppocr_native_b200 import cuda
from test_block_ops import DTYPES, Q4, Attn, half_step, norm_check

gpu = pytest.mark.gpu
CSRC = Path(cuda.__file__).resolve().parent / "csrc"


# ---------------------------------------------------------------- the 4-bit product

def test_q4_clusters_have_started_before_remote_stores():
    # a block may write into another's shared memory only once that block runs: each
    # kernel arrives at the cluster's barrier before its first load, and the join waits
    # for it before its first remote store
    join = (CSRC / "q4.cuh").read_text().split("void join(")[1]
    assert 0 <= join.find("cluster_wait();") < join.find("peer_store(part")
    for name in ("k_q4.cu", "k_q4_int.cu"):
        kernel = (CSRC / name).read_text().split("__global__")[1]
        assert 0 <= kernel.find("if (a.ks > 1) cluster_arrive();") < kernel.find("in.begin(a, at);"), name


@gpu
@pytest.mark.parametrize("xt,m,k,n,group", [("f32", 1, 20000, 40, 32), ("f32", 2, 70000, 20, 128), ("f32", 5, 9000, 64, 64),
                                            ("f16", 16, 16384, 256, 64), ("e4m3", 9, 30000, 30, 128)])
def test_q4_clusters_beside_other_work(cuda_mod, xt, m, k, n, group):
    # the blocks of a cluster start apart while other launches come and go
    a = Q4(xt, "f32", m, k, n, group, seed=31)
    a.call()
    a.check()
    want = a.y.clone()
    other, big = torch.cuda.Stream(), torch.zeros(1 << 22, device="cuda")
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(other):
            big.add_(1.0)
        a.y.zero_()
        a.call()
        assert torch.equal(a.y, want)


def q4_close(a):
    """As Q4.check for f32 outputs, with errors that add up as the root of their number.
    S is the root of the sum of the products' squares; partial sums of terms of any sign
    stay below 3 S or so. A group's sum takes at most 8 instructions of 16 k, each cutting at
    most 2^-23 of it, all toward zero: 24 S 2^-23 over the groups, whose signs differ. Each of
    the G groups' additions rounds 2^-24 of at most 3 S, independently: sqrt(G) S 2^-23. Eight
    more roundings end it (joins, scales, the bias, a product of x and its scale)."""
    _, _, _, m, k, n, group, _ = a.args
    q = torch.stack([a.w & 15, a.w >> 4], 2).flatten(1)[:, :k].double()
    each = torch.arange(k, device="cuda") // group
    w = (q - (a.zeros.double()[:, each] if a.zeros is not None else 8)) * a.scales.double()[:, each]
    want, squares = a.value @ w.T, a.value.square() @ w.T.square()
    bias = a.bias.double() if a.bias is not None else torch.zeros(n, dtype=torch.float64, device="cuda")
    tol = 2.0 ** -23 * (squares.sqrt() * (24 + math.sqrt(w.shape[1] / min(group, 128)) + 8) + (want + bias).abs())
    off = (a.y.double() - want - bias).abs()
    assert bool((off <= tol).all()), float((off / tol).nan_to_num(math.inf).max())
    return tol


@gpu
@pytest.mark.parametrize("m,k,n,group", [(1, 120, 360, 32), (2, 64, 170, 64), (3, 1000, 777, 32), (5, 257, 100, 128),
                                         (10, 4096, 64, 64), (11, 640, 130, 64), (32, 2049, 40, 32), (1, 8192, 300, 128),
                                         (2, 8192, 300, 64), (4, 20000, 70, 128), (9, 9000, 40, 64)])
@pytest.mark.parametrize("zeros", [False, True])
def test_q4_f32_rows_keep_24_bits(cuda_mod, m, k, n, group, zeros):
    a = Q4("f32", "f32", m, k, n, group, zeros, scale_type="f32", seed=k)
    a.bias.zero_()
    a.call()
    tol = q4_close(a)
    # the bound notices 16 bits in place of 24
    cut = (a.x.view(torch.int32) & -256).view(torch.float32).double()
    q = torch.stack([a.w & 15, a.w >> 4], 2).flatten(1)[:, :k].double()
    each = torch.arange(k, device="cuda") // group
    w = (q - (a.zeros.double()[:, each] if zeros else 8)) * a.scales.double()[:, each]
    assert bool((((cut - a.value) @ w.T).abs() > tol).any())


@gpu
@pytest.mark.parametrize("xt,m,k,n", [("f32", 1, 512, 400), ("f32", 2, 512, 400), ("f32", 1, 5000, 90), ("f32", 2, 5000, 90),
                                      ("f32", 3, 700, 90), ("f16", 1, 4129, 8203), ("bf16", 1, 4129, 8203),
                                      ("f16", 2, 4129, 8203), ("bf16", 2, 4129, 8203), ("e4m3", 1, 4129, 8203),
                                      ("f16", 1, 8257, 8203), ("bf16", 1, 8257, 8203), ("e4m3", 1, 8257, 8203)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("far", [10, 14, 20, 30])
@pytest.mark.parametrize("hidden", ["weight", "scale"])
def test_q4_one_value_far_above_the_rest(cuda_mod, xt, m, k, n, group, far, hidden):
    # a channel that its weights take out again, by their zero point or their group's
    # small scale: the others' sum keeps its bits
    if xt in ("f16", "e4m3") and far > 10:
        pytest.skip("beyond the type")
    a = Q4(xt, "f32", m, k, n, group, True, scale_type="f32", seed=k + far)
    a.bias.zero_()
    x = a.x.float()
    if xt == "e4m3":
        x *= 2.0 ** -8
        x[:, 77] = 256.0
    else:
        x[:, 77] = 1.7 * 2.0 ** far
    a.x = x.to(a.x.dtype)
    a.value = a.x.double() * (a.x_scales.double() if xt == "e4m3" else 1)
    if hidden == "weight":
        z = a.zeros[:, 77 // group]
        a.w[:, 77 // 2] = (a.w[:, 77 // 2] & 15) | (z << 4)
    else:
        a.scales[:, 77 // group] = 2.0 ** -far * 2.0 ** -6
    a.call()
    q4_close(a)


@gpu
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("group,zeros,x_group", [(128, False, 0), (128, True, 0), (64, True, 0), (32, True, 0), (96, False, 0),
                                                 (64, True, 64)])
def test_q4_one_row_of_very_many_weights(cuda_mod, xt, group, zeros, x_group):
    # odd sizes beyond 2^26 weights, a NaN, and rows of w side by side
    if x_group and xt != "e4m3":
        pytest.skip("scales of x belong to e4m3")
    for pad in (3, 0):
        a = Q4(xt, "f32", 1, 8257, 8203, group, zeros, x_group=x_group, w_pad=pad, seed=19)
        a.call()
        a.check()
        q4_close(a)
        x = a.x.float()
        x[0, 4001] = math.nan
        a.x = x.to(a.x.dtype)
        a.call()
        assert bool(a.y.isnan().all())


@gpu
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("k,group", [(300, 32), (5000, 128)])
def test_q4_f32_rows_of_every_magnitude(cuda_mod, m, k, group):
    # magnitudes spread over 2^39: what lies below 2^-62 of a slice's largest may go, no more
    for top in (2.0 ** 100, 2.0 ** -110, 1.0):
        a = Q4("f32", "f32", m, k, 70, group, scale_type="f32", seed=k)
        a.bias.zero_()
        a.x = torch.ldexp(a.x.clamp(-1, 1), torch.randint(-39, 1, a.x.shape, device="cuda")) * top
        for hide in (False, True):
            if hide:  # the largest taken out by its weight, the rest keep what they have
                a.x[:, 40] = 3.0 * top
                a.w[:, 20] = (a.w[:, 20] & 0xF0) | a.zeros[:, 40 // group]
            a.value = a.x.double()
            a.call()
            q = torch.stack([a.w & 15, a.w >> 4], 2).flatten(1)[:, :k].double()
            each = torch.arange(k, device="cuda") // group
            w = (q - a.zeros.double()[:, each]) * a.scales.double()[:, each]
            # q4_close's bound, and half a step of each x
            want, squares = a.value @ w.T, a.value.square() @ w.T.square()
            tol = 2.0 ** -23 * (squares.sqrt() * (32 + math.sqrt(k / min(group, 128))) + want.abs())
            tol = tol + 3.0 * top * 2.0 ** -62 * w.abs().sum(1) + 2.0 ** -149 * k
            assert bool(((a.y.double() - want).abs() <= tol).all())


# ---------------------------------------------------------------- the norm

def norm_run(t, x, r, gamma, eps, group):
    rows, c = x.shape
    s, y = torch.empty_like(x), torch.empty(rows, c, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, -(-c // group) if group else 1, device="cuda")
    cuda.rms_norm_e4m3(cuda.RmsNormShape(t, rows, c, group, eps), x.data_ptr(), r.data_ptr() if r is not None else None,
                       gamma.data_ptr(), s.data_ptr(), y.data_ptr(), scales.data_ptr(),
                       torch.cuda.current_stream().cuda_stream)
    norm_check(t, x, r, gamma, eps, group, s, y, scales)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("c", [100, 500, 1001, 1024, 2047, 4096, 8192, 20000, 32768])
def test_norm_rows_far_from_one(cuda_mod, t, group, c):
    # squares that f32 does not hold, alone or summed; rows of ordinary size among them
    g = torch.Generator("cuda").manual_seed(c)
    sizes = [1e18, 1.0, 1.8e19, 3e30, 1e38, 1e-15, 1e-19, 1e-23, 1e-30, 1e-35, 1.0, 6e-13, 3e-13, 1e-12, 2e-11, 1e15, 3e14, 1e16]
    x = torch.randn(len(sizes), c, generator=g, device="cuda") * torch.tensor(sizes, device="cuda")[:, None]
    x[0] = 1e18
    x = x.clamp(-2e38, 2e38).to(DTYPES[t])
    r = torch.zeros_like(x)
    r[1] = 1
    gamma = 0.5 + 0.5 * torch.rand(c, generator=g, device="cuda")
    norm_run(t, x, r, gamma, 0.0, group)
    norm_run(t, x, None, gamma, 0.0, group)
    norm_run(t, x, r, gamma, 1e-6, group)
    norm_run(t, x, r, gamma, 1e-37, group)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("c", [120, 1003, 4096])
def test_norm_rows_of_two_sizes(cuda_mod, t, c):
    # one thread's channels far above, or below, all the others'; runs of zeros
    g = torch.Generator("cuda").manual_seed(c)
    for size in (1e25, 1e-25):
        x = torch.randn(9, c, generator=g, device="cuda")
        x[1:4, 40:48] *= size
        x[4:6, 5] *= size
        x[6:8] = 0
        x[7:, 64:72] = size
        norm_run(t, x.to(DTYPES[t]), None, torch.ones(c, device="cuda"), 1e-6, 0)
        norm_run(t, x.to(DTYPES[t]), None, torch.ones(c, device="cuda"), 1e-6, 32)


# ---------------------------------------------------------------- attention

@gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("steps", [False, True])
@pytest.mark.parametrize("sign", [-1, 1])
def test_attention_scores_near_the_largest_number(cuda_mod, t, d, steps, sign):
    # finite scores that their conversion to powers of two takes past the largest number:
    # equal ones weigh the same, and one far above the others has all the weight
    lens = [(2, 600), (1, 77)] if steps else [(300, 300), (77, 77)]
    a = Attn(t, lens, 4, 2, d, 50, 0, 3, seed=41, interleaved=False, room=650, scale=1.0)
    a.q.zero_(), a.k.zero_()
    a.q[..., 0] = 1
    a.k[..., 0] = sign * 3e38
    a.call()

    def weighted(weight):
        # weight(j): a key's, by its place in the lane
        at = 0
        for (nq, nk), begin in zip(a.lens, a.begin):
            p, j = torch.arange(nq, device="cuda")[:, None] + nk - nq, torch.arange(nk, device="cuda")[None]
            seen = ((j <= p) & ((j >= p - 50) | (j < 3))).double() * weight(j)
            v = a.v[begin:begin + nk].double().repeat_interleave(2, 1)
            want = torch.einsum("ij,jhd->ihd", seen / seen.sum(1, keepdim=True), v)
            mags = torch.einsum("ij,jhd->ihd", seen / seen.sum(1, keepdim=True), v.abs())
            # weights (exact ones, their sum, a quotient) and the products' sum, then the output's rounding
            tol = mags * (half_step(t) + (nk + 8) * 2.0 ** -23) + half_step(t) * want.abs()
            assert bool(((a.out[at:at + nq].double() - want).abs() <= tol).all())
            at += nq

    weighted(lambda j: torch.ones_like(j).double())
    # every seventh key above the rest by more than any weight holds
    for begin, (_, nk) in zip(a.begin, a.lens):
        j = torch.arange(nk, device="cuda")
        a.k[begin:begin + nk, :, 0] = torch.where(j % 7 == 0, 3e38, 2.9e38 if sign > 0 else 3.2e38)[:, None].to(a.k.dtype) * sign
    a.call()
    weighted(lambda j: (j % 7 == 0).double())


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("what", ["key", "value"])
def test_attention_one_early_key_that_is_no_number(cuda_mod, t, what):
    # every later row sees it and is done again: a NaN score ends such a row at once, an
    # infinite value takes the plain loop's time (a key at a time: 199 ms here)
    n, heads, d = 4000, 8, 64
    a = Attn(t, [(n, n)], heads, 2, d, -1, 0, 0, seed=43, interleaved=False)
    times = []
    for bad in (False, True):
        if bad and what == "key":
            a.k[5, :, 3] = math.nan
        if bad and what == "value":
            a.v[5, :, 3] = math.inf
        a.call()
        torch.cuda.synchronize()
        first, last = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        first.record()
        a.call()
        last.record()
        torch.cuda.synchronize()
        times.append(first.elapsed_time(last))
    a.check()
    if what == "key":
        assert bool(a.out[5:].isnan().all())
    else:
        assert bool((a.out[5:, :, 3] == math.inf).all()) and bool(a.out[..., :3].isfinite().all())
    assert times[1] <= (60 if what == "value" else 10), times


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[(300, 300), (1, 1), (77, 77)], [(1, 500), (2, 90)]])
def test_attention_broadcast_inputs(cuda_mod, t, lens):
    # one head, or one row, that stands for all: strides of zero
    room = 510 if lens[0][0] == 1 else 0
    for what in ("heads", "rows", "queries"):
        a = Attn(t, lens, 4, 2, 64, 60, 5, 2, seed=53, interleaved=False, room=room, pad=2)
        if what == "heads":
            a.k, a.v = a.k[:, :1].expand(-1, 2, -1), a.v[:, :1].expand(-1, 2, -1)
        elif what == "rows":
            a.k, a.v = a.k[:1].expand(a.k.shape[0], -1, -1), a.v[:1].expand(a.v.shape[0], -1, -1)
        else:
            a.q = a.q[:1, :1].expand(a.q.shape[0], 4, -1)
        a.call()
        a.check()


# ---------------------------------------------------------------- buffers

@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("lens", [[(300, 300), (1, 1), (77, 77)], [(1, 500), (2, 90)]])
def test_attention_page_locked_buffers(cuda_mod, t, d, lens):
    a = Attn(t, lens, 4, 2, d, 60, 5, 2, seed=51, interleaved=False, room=510 if lens[0][0] == 1 else 0, pad=2)
    host = {k: getattr(a, k).contiguous().cpu().pin_memory() for k in ("q", "k", "v", "out", "offsets", "k_begin", "k_len")}
    strides = {k + "_strides": host[k].stride()[:2] for k in ("q", "k", "v", "out")}
    cuda.attention_window(a.shape(**strides), *(host[k].data_ptr() for k in ("q", "k", "v", "out", "offsets", "k_begin", "k_len")),
                          torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    a.out.copy_(host["out"])
    a.check()


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_norm_and_q4_page_locked_buffers(cuda_mod, t):
    stream = torch.cuda.current_stream().cuda_stream
    for c in (256, 101):
        x, r = (torch.randn(30, c).to(DTYPES[t]).pin_memory() for _ in range(2))
        s, y = torch.empty_like(x).pin_memory(), torch.empty(30, c, dtype=torch.uint8).pin_memory()
        gamma, scales = torch.rand(c).pin_memory(), torch.empty(30, 1).pin_memory()
        cuda.rms_norm_e4m3(cuda.RmsNormShape(t, 30, c, 0, 1e-6), x.data_ptr(), r.data_ptr(), gamma.data_ptr(), s.data_ptr(),
                           y.data_ptr(), scales.data_ptr(), stream)
        torch.cuda.synchronize()
        norm_check(t, x.cuda(), r.cuda(), gamma.cuda(), 1e-6, 0, s.cuda(), y.cuda(), scales.cuda())
    for m in (1, 2, 16):
        a = Q4(t, "f32", m, 500, 300, 64, seed=52)
        a.call()
        want, dev = a.y.clone(), {k: getattr(a, k) for k in ("x", "w", "scales", "zeros", "bias", "y")}
        for k, v in dev.items():
            setattr(a, k, v.cpu().pin_memory())
        a.y.zero_()
        a.call()
        torch.cuda.synchronize()
        assert torch.equal(a.y.cuda(), want)


def test_columns_of_one_buffer_do_not_overlap():
    # rows side by side in a wider buffer share no element; one element shared is refused
    p = 1 << 20

    def outcome(call):
        with pytest.raises(cuda.PpocrError) as e:
            call()
        return "overlap" in str(e.value)

    wide = [(512, 64)] * 4  # q, k, v and out of 2 heads of 64 in rows of 512 elements

    def attention(q, k, v, out, **kw):
        shape = cuda.AttentionShape(**({"type": "f16", "lanes": 1, "heads": 2, "kv_heads": 2, "head_dim": 64, "q_rows": 9,
                                        "kv_rows": 9, "scale": 1.0, "q_strides": wide[0], "k_strides": wide[1],
                                        "v_strides": wide[2], "out_strides": wide[3]} | kw))
        cuda.attention_window(shape, p + 2 * q, p + 2 * k, p + 2 * v, p + 2 * out, p << 4)

    assert not outcome(lambda: attention(0, 128, 256, 384))
    assert not outcome(lambda: attention(384, 256, 128, 0))
    assert outcome(lambda: attention(0, 128, 256, 383)) and outcome(lambda: attention(0, 128, 256, 385))
    assert outcome(lambda: attention(0, 128, 256, 384, out_strides=(1024, 64)))
    assert outcome(lambda: attention(0, 512 * 4 + 384 + 64, 256, 384))

    def norm(x, residual, sum, **kw):
        shape = cuda.RmsNormShape(**({"type": "f16", "rows": 7, "channels": 100, "x_row": 300, "residual_row": 300,
                                      "sum_row": 300} | kw))
        cuda.rms_norm_e4m3(shape, p + 2 * x, p + 2 * residual, p << 5, p + 2 * sum, p << 6, p << 7)

    assert not outcome(lambda: norm(0, 100, 200)) and not outcome(lambda: norm(200, 100, 0))
    assert outcome(lambda: norm(0, 100, 199)) and outcome(lambda: norm(0, 100, 201)) and outcome(lambda: norm(0, 100, 200, sum_row=299))

    def q4(x, y, **kw):
        shape = cuda.MatvecQ4Shape(**({"x_type": "f16", "y_type": "f16", "scale_type": "f16", "rows": 3, "k": 64, "n": 32,
                                       "group": 32, "x_row": 96, "y_row": 96} | kw))
        cuda.matvec_q4(shape, p + 2 * x, None, p << 5, p << 6, None, None, p + 2 * y)

    assert not outcome(lambda: q4(0, 64)) and not outcome(lambda: q4(32, 0)) and not outcome(lambda: q4(96 + 32, 0))
    assert outcome(lambda: q4(0, 63)) and outcome(lambda: q4(0, 65)) and outcome(lambda: q4(0, 64, y_type="f32"))


@gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_outputs_beside_inputs_in_one_buffer(cuda_mod, t):
    n, h, d, size = 200, 4, 32, torch.finfo(DTYPES[t]).bits // 8
    a = Attn(t, [(n, n)], h, h, d, 40, 3, 1, seed=61, interleaved=False)
    rows = torch.full((n, 4 * h, d), 7.0, device="cuda").to(DTYPES[t])
    rows[:, :h], rows[:, h:2 * h], rows[:, 2 * h:3 * h] = a.q, a.k, a.v
    a.q, a.k, a.v, a.out = (rows[:, i * h:(i + 1) * h] for i in range(4))
    before = rows[:, :3 * h].clone()
    a.call()
    a.check()
    assert torch.equal(rows[:, :3 * h], before)
    c = 120
    wide = torch.randn(50, 3 * c, device="cuda").to(DTYPES[t])
    x, r, gamma = wide[:, :c].clone(), wide[:, c:2 * c].clone(), torch.rand(c, device="cuda")
    y, scales = torch.empty(50, c, dtype=torch.uint8, device="cuda"), torch.empty(50, 1, device="cuda")
    cuda.rms_norm_e4m3(cuda.RmsNormShape(t, 50, c, 0, 1e-6, 3 * c, 3 * c, 3 * c), wide.data_ptr(), wide.data_ptr() + c * size,
                       gamma.data_ptr(), wide.data_ptr() + 2 * c * size, y.data_ptr(), scales.data_ptr(),
                       torch.cuda.current_stream().cuda_stream)
    norm_check(t, x, r, gamma, 1e-6, 0, wide[:, 2 * c:], y, scales)
    assert torch.equal(wide[:, :c], x) and torch.equal(wide[:, c:2 * c], r)
    for m in (1, 8):
        b = Q4(t, t, m, 256, 96, 32, seed=62)
        b.call()
        both = torch.empty(m, 352, device="cuda").to(DTYPES[t])
        both[:, :256] = b.x
        want, b.x, b.y = b.y, both, both[:, 256:]
        b.call(x_row=352, y_row=352)
        assert torch.equal(both[:, 256:], want)
