"""8-bit rows, weights and products against the same in 64 bits: one row to many, odd sizes, slices of wider tensors, zeros,
infinities, the borders of the scales; a run of them together as a feed-forward uses them; and captured runs."""
import math

import pytest
import torch

import fp8_util as fu

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from tiny_llm_b200 import ops
    return ops


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def rows8(ops, x):
    out = ops.fp8_rows(x.shape[0], x.shape[1], DEV)
    ops.quantize_fp8(x, *out)
    return out


def weight8(ops, w):
    out = ops.fp8_weight(w.shape[0], w.shape[1], DEV)
    ops.quantize_weight_fp8(w, *out)
    return out


def same(got, want):
    return bool(((got.double() == want) | (torch.isnan(got.double()) & torch.isnan(want))).all())


def spread(g, m, k):
    """Rows whose groups differ by many powers of two, with zeros among them."""
    x = randn(g, m, k) * torch.exp2(torch.randint(-20, 20, (m, fu.groups(k)), generator=g, device=DEV).float()).repeat_interleave(128, 1)[:, :k]
    x[torch.rand(m, k, generator=g, device=DEV) < 0.2] = 0
    return x


# ---------------------------------------------------------------------------------------------- rows and weights


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (7, 129), (33, 2000), (5, 514), (300, 1030), (2, 14336), (1000, 136)])
def test_rows_are_the_nearest_8_bit_values(ops, m, k, dtype):
    g = rng(m * 31 + k)
    wide = spread(g, m, k + 5).to(dtype)
    for x in (wide[:, :k].contiguous(), wide[:, :k], wide[:, 5:]):
        room = torch.full((m, -(-k // 16) * 16 + 16), 7, dtype=torch.uint8, device=DEV)
        scales = torch.full((m, fu.groups(k) + 3), 7, dtype=torch.uint8, device=DEV)
        out, sc = room.view(ops.FP8)[:, :k], scales.view(ops.FP8_SCALE)[:, : fu.groups(k)]
        ops.quantize_fp8(x, out, sc)
        want, ws = fu.quantize_rows(x)
        assert same(out, want) and same(sc, ws)
        assert bool((room[:, k:] == 7).all()) and bool((scales[:, fu.groups(k):] == 7).all())   # what lies behind stays


def test_scales_at_their_borders(ops):
    """Largest magnitudes at and next to 448 times powers of two, the smallest and largest floats, zeros, infinities, NaN."""
    up = torch.tensor(448.0).nextafter(torch.tensor(1e9)).item()
    edges = [448.0, up, 447.0, 1.75, 1.75 * 2.0 ** -100, 0.0, -0.0, 2.0 ** -149, 2.0 ** -126, 448 * 2.0 ** -126, up * 2.0 ** -126,
             3.4028234663852886e38, -3.4028234663852886e38, math.inf, -math.inf, math.nan, 464.0, 1.0, 2.0 ** -10]
    x = torch.zeros(len(edges), 300, device=DEV)
    x[:, 1] = 2.0 ** -9 * 1.5                       # beside a 1 it is a tie between two 8-bit values or far below them
    x[:, 290] = 1.0
    for i, e in enumerate(edges):
        x[i, 77] = e
    out, sc = rows8(ops, x)
    want, ws = fu.quantize_rows(x)
    assert same(sc, ws) and same(out, want)
    assert torch.isnan(sc.float()[13:16, 0]).all() and bool((out.float()[13:16, :128] == 0).all()) and bool((sc.float()[:, 2] == 2.0 ** -8).all())
    blocks = torch.zeros(128 * len(edges), 130, device=DEV)
    blocks[::128, 0] = x[:, 77]
    data, scales = weight8(ops, blocks)
    want, ws = fu.quantize_weight(blocks)
    assert same(scales, ws) and same(data, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (127, 129), (128, 128), (300, 1000), (257, 4099), (2560, 2048)])
def test_weights_are_the_nearest_8_bit_values(ops, n, k, dtype):
    g = rng(n + k)
    wide = (randn(g, n, k + 3) * torch.exp2(torch.randint(-9, 9, (n, 1), generator=g, device=DEV).float())).to(dtype)
    for w in (wide[:, :k].contiguous(), wide[:, 3:]):
        data, scales = weight8(ops, w)
        want, ws = fu.quantize_weight(w)
        assert same(data, want) and same(scales, ws)


@pytest.mark.parametrize("m,k", [(1, 64), (3, 130), (8, 2048), (5, 4097), (40, 1000), (2, 20000), (2, 40000), (700, 512)])
def test_normed_rows(ops, m, k):
    """The mean of squares and the two products in 32 bits: at most k / 512 + 20 roundings of 2^-24."""
    g = rng(m + k)
    x, w = spread(g, m + 2, k), 1 + 0.3 * randn(g, k)
    x[m + 1] = 0
    idx = torch.randperm(m + 2, generator=g, device=DEV)[: m + 1].to(torch.int32)
    y = w.double() * x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-5)
    off = y.abs() * (k / 512 + 20) * 2.0 ** -24
    out = ops.fp8_rows(m + 2, k, DEV)
    ops.rms_norm_fp8(x, w, 1e-5, *out)
    assert fu.between_roundings(*out, y, off) and bool((out[0].float()[m + 1] == 0).all())
    some = ops.fp8_rows(m + 1, k, DEV)
    ops.rms_norm_fp8(x, w, 1e-5, *some, rows=idx)
    assert torch.equal(some[0].view(torch.uint8), out[0].view(torch.uint8)[idx.long()]) and torch.equal(some[1].view(torch.uint8), out[1].view(torch.uint8)[idx.long()])


# ---------------------------------------------------------------------------------------------- products


SHAPES = [(1, 1, 1), (1, 2560, 2048), (2, 130, 300), (5, 1000, 129), (16, 64, 4096), (17, 4100, 520), (33, 700, 1152), (64, 512, 3584),
          (65, 129, 700), (100, 4096, 640), (127, 300, 257), (128, 384, 128), (129, 128, 1000), (200, 1000, 1520), (257, 2000, 400),
          (400, 5000, 384), (1000, 333, 260), (1500, 2304, 512), (2100, 4000, 200)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_are_near_64_bits(ops, m, n, k):
    g = rng(m + 3 * n + 7 * k)
    a, w = rows8(ops, spread(g, m, k)), weight8(ops, randn(g, n, k))
    w[1].mul_(torch.rand(w[1].shape, generator=g, device=DEV) + 0.5)        # scales of any value
    want, off = fu.product(*a, *w)
    full = torch.full((m, n + 5), 7.0, device=DEV)
    for out in (torch.empty(m, n, device=DEV), full[:, :n], torch.full((m, n + 3), 7.0, device=DEV)[:, 3:]):
        ops.linear_fp8(*a, *w, out)
        assert bool(((out - want).abs() <= off + 2.0 ** -24 * want.abs()).all())
    assert bool((full[:, n:] == 7.0).all())
    short = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    ops.linear_fp8(*a, *w, short)
    assert bool(((short.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all())
    stream = randn(g, m, n)
    acc = stream.clone()
    ops.linear_fp8(*a, *w, acc, accumulate=True)
    assert bool(((acc - (stream + want)).abs() <= off + 2.0 ** -24 * ((stream + want).abs() + want.abs() + off)).all())
    again = torch.empty(m, n, device=DEV)
    ops.linear_fp8(*a, *w, again)
    assert torch.equal(again, full[:, :n])                                   # no order of sums changes from call to call
    ops.check_status()


@pytest.mark.parametrize("m", [3, 40, 150, 600])
def test_rows_that_are_not_finite_spoil_no_other_row(ops, m):
    g = rng(m)
    n, k = 700, 1000
    x = randn(g, m, k)
    x[1, 5], x[2, 999] = math.inf, math.nan
    a, w = rows8(ops, x), weight8(ops, randn(g, n, k))
    out = torch.empty(m, n, device=DEV)
    ops.linear_fp8(*a, *w, out)
    clean = x.clone()
    clean[1:3] = 0
    want, off = fu.product(*rows8(ops, clean), *w)
    assert bool(torch.isnan(out[1:3]).all())
    keep = [i for i in range(m) if i not in (1, 2)]
    assert bool(((out - want).abs() <= off + 2.0 ** -24 * want.abs())[keep].all())


def gated_weight(ops, g, i, k):
    blocks = fu.groups(i)
    w = torch.zeros(2, blocks * 128, k, device=DEV)
    w[:, :i] = randn(g, 2, i, k) / math.sqrt(k)
    return weight8(ops, w.view(2, blocks, 128, k).transpose(0, 1).reshape(2 * blocks * 128, k).contiguous())


@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("relu", 0.0), ("clamped", 1.5), ("gelu_tanh", 0.0)])
@pytest.mark.parametrize("m,i,k", [(1, 5632, 2048), (3, 1, 130), (16, 128, 512), (17, 1000, 300), (40, 300, 2000), (64, 2050, 256), (70, 200, 1111),
                                   (128, 640, 384), (129, 129, 500), (300, 1000, 640), (1300, 777, 260)])
def test_gated_products(ops, m, i, k, act, limit):
    g = rng(m + i + k)
    a, w = rows8(ops, 2 * randn(g, m, k)), gated_weight(ops, g, i, k)
    want, off = fu.gated(*a, *w, i, act, limit)
    wide = torch.full((m, i + 3), 7.0, dtype=torch.bfloat16, device=DEV)
    for out in (torch.empty(m, i, dtype=torch.bfloat16, device=DEV), wide[:, :i]):
        ops.linear_swiglu_fp8(*a, *w, out, act=act, limit=limit)
        assert bool(((out.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all())
    assert bool((wide[:, i:] == 7.0).all())
    room = torch.full((m, -(-i // 16) * 16 + 16), 7, dtype=torch.uint8, device=DEV)
    scales = torch.full((m, fu.groups(i) + 3), 7, dtype=torch.uint8, device=DEV)
    out, sc = room.view(ops.FP8)[:, :i], scales.view(ops.FP8_SCALE)[:, : fu.groups(i)]
    ops.linear_swiglu_fp8(*a, *w, out, sc, act=act, limit=limit)
    assert fu.between_roundings(out, sc, want, off)
    assert bool((room[:, i:] == 7).all()) and bool((scales[:, fu.groups(i):] == 7).all())
    ops.check_status()


@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("relu", 0.0), ("clamped", 1.5), ("gelu_tanh", 0.0)])
@pytest.mark.parametrize("m", [3, 100, 2400])
def test_gates_beyond_32_bits(ops, m, act, limit):
    """Gate sums of 2^135 (infinite in 32 bits), 2^75, -2^75 and 2^-140 (next to nothing) beside up sums of 128.  The sums are exact, so
    what is left is the gate's 2^-20 and the rounding to 8 bits of mantissa."""
    a = rows8(ops, torch.ones(m, 128, device=DEV))
    w = torch.ones(4, 2, 128, 128, device=DEV)
    w[2, 0] = -1.0
    w = weight8(ops, w.view(1024, 128))
    w[1][0::2] *= torch.tensor([2.0 ** 120, 2.0 ** 68, 2.0 ** 68, 2.0 ** -118], device=DEV)[:, None] * 2.0 ** 8
    want, _ = fu.gated(*a, *w, 512, act, limit)
    out = torch.empty(m, 512, dtype=torch.bfloat16, device=DEV)
    ops.linear_swiglu_fp8(*a, *w, out, act=act, limit=limit)
    beyond = want.abs() > 2.0 ** 128
    assert bool(beyond[:, :128].all()) == (act != "clamped") and not bool(beyond[:, 128:].any())
    assert bool((out[beyond] == math.inf).all())
    got, want = out.double()[~beyond], want[~beyond]
    assert bool(((got - want).abs() <= (2.0 ** -8 + 2.0 ** -19) * want.abs() + 2.0 ** -126).all())
    ops.check_status()


# ---------------------------------------------------------------------------------------------- together


@pytest.mark.parametrize("m", [1, 9, 100, 513])
def test_a_feed_forward_in_8_bits(ops, m):
    """Norm, gate and up, down into the stream, one kernel each, on another stream than the default one and captured: the graph
    does with new rows what the calls do.  Against the same chain in 64 bits from the kernel's own 8-bit rows."""
    g = rng(m)
    h, i = 520, 1000
    x, norm = randn(g, m, h), 1 + 0.2 * randn(g, h)
    gate_up, down = gated_weight(ops, g, i, h), weight8(ops, randn(g, h, i) / math.sqrt(i))
    y, mid, out = ops.fp8_rows(m, h, DEV), ops.fp8_rows(m, i, DEV), x.clone()

    def chain():
        ops.rms_norm_fp8(x, norm, 1e-5, *y)
        ops.linear_swiglu_fp8(*y, *gate_up, *mid)
        ops.linear_fp8(*mid, *down, out, accumulate=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    want, off = fu.product(*mid, *down)
    assert bool(((out - (x + want)).abs() <= off + 2.0 ** -23 * ((x + want).abs() + want.abs() + off)).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    fresh = randn(g, m, h)
    for rows in (x.clone(), fresh):
        x.copy_(rows)
        out.copy_(rows)
        graph.replay()
        replayed = out.clone()
        out.copy_(rows)
        chain()
        assert torch.equal(out, replayed)
    ops.check_status()


@pytest.mark.parametrize("m", [1, 50, 300])
def test_a_weight_may_be_made_right_before_it_is_read(ops, m):
    """Products begin to read their weight while earlier launches run; the kernel that makes an 8-bit weight does not let them."""
    g = rng(m)
    n, k = 4096, 4096
    a, w = rows8(ops, randn(g, m, k)), [randn(g, n, k) for _ in range(4)]
    room, out = ops.fp8_weight(n, k, DEV), [torch.empty(m, n, device=DEV) for _ in w]
    for x, o in zip(w, out):
        ops.quantize_weight_fp8(x, *room)
        ops.linear_fp8(*a, *room, o)
    for x, o in zip(w, out):
        want, off = fu.product(*a, *weight8(ops, x))
        assert bool(((o - want).abs() <= off + 2.0 ** -24 * want.abs()).all())


def test_no_rows(ops):
    g = rng(0)
    w = weight8(ops, randn(g, 256, 128))
    a = ops.fp8_rows(0, 128, DEV)
    before = ops.launches
    ops.quantize_fp8(torch.empty(0, 128, device=DEV), *a)
    ops.linear_fp8(*a, *w, torch.empty(0, 256, device=DEV))
    ops.linear_swiglu_fp8(*a, *w, torch.empty(0, 128, dtype=torch.bfloat16, device=DEV))
    assert ops.launches == before


# ---------------------------------------------------------------------------------------------- calls


def calls(ops, m, n, k):
    """Every operator once, as (what it leaves, the call)."""
    g = rng(m + n + k)
    x, w, norm = randn(g, m, k), randn(g, n, k), 1 + 0.1 * randn(g, k)
    a, w8, gu = rows8(ops, x), weight8(ops, w), gated_weight(ops, g, n, k)
    rows, rows_b, weight = ops.fp8_rows(m, k, DEV), ops.fp8_rows(m, k, DEV), ops.fp8_weight(n, k, DEV)
    f32, bf16, acc, wide = torch.empty(m, n, device=DEV), torch.empty(m, n, dtype=torch.bfloat16, device=DEV), torch.zeros(m, n, device=DEV), torch.zeros(m, n + 9, device=DEV)
    h, h8 = torch.empty(m, n, dtype=torch.bfloat16, device=DEV), ops.fp8_rows(m, n, DEV)
    idx = torch.arange(m, dtype=torch.int32, device=DEV).flip(0)
    return [(rows, lambda: ops.quantize_fp8(x, *rows)), (rows, lambda: ops.quantize_fp8(x.bfloat16(), *rows)), (weight, lambda: ops.quantize_weight_fp8(w, *weight)),
            (rows_b, lambda: ops.rms_norm_fp8(x, norm, 1e-5, *rows_b)), (rows_b, lambda: ops.rms_norm_fp8(x, norm, 1e-5, *rows_b, rows=idx)),
            ((f32,), lambda: ops.linear_fp8(*a, *w8, f32)), ((bf16,), lambda: ops.linear_fp8(*a, *w8, bf16)),
            ((acc,), lambda: ops.linear_fp8(*a, *w8, acc.zero_(), accumulate=True)), ((wide,), lambda: ops.linear_fp8(*a, *w8, wide[:, 4: 4 + n])),
            ((h,), lambda: ops.linear_swiglu_fp8(*a, *gu, h)), (h8, lambda: ops.linear_swiglu_fp8(*a, *gu, *h8, act="clamped", limit=2.0)),
            (h8, lambda: ops.linear_swiglu_fp8(*a, *gu, *h8, act="gelu_tanh"))]


@pytest.mark.parametrize("m,n,k", [(1, 256, 128), (2, 130, 200), (200, 300, 77)])
def test_calls_through_the_interpreter_do_the_same(ops, monkeypatch, m, n, k):
    for left, call in calls(ops, m, n, k):
        call()                                                       # (the first one loads what there is)
        assert ops._fp8_native, "the calls' extension was not built"
        before = ops.launches
        call()
        assert ops.launches == before + 1
        want = [t.contiguous().view(torch.uint8).clone() for t in left]
        monkeypatch.setattr(ops, "_fp8_native", False)
        call()
        assert ops.launches == before + 2
        monkeypatch.undo()
        assert all(torch.equal(t.contiguous().view(torch.uint8), v) for t, v in zip(left, want))


def test_refused_calls_launch_nothing(ops):
    g = rng(0)
    x, a, w = randn(g, 4, 256), ops.fp8_rows(4, 256, DEV), weight8(ops, randn(g, 300, 256))
    ops.quantize_fp8(x, *a)
    out, before = torch.full((4, 300), 7.0, device=DEV), ops.launches
    for call in (lambda: ops.linear_fp8(*a, *w, out[:, :299]), lambda: ops.linear_fp8(a[0][:, 16:], a[1], *w, out), lambda: ops.linear_fp8(*a, *w, out.cpu()),
                 lambda: ops.linear_fp8(a[0], a[1].float(), *w, out), lambda: ops.linear_fp8(*a, w[0], w[1][:2], out), lambda: ops.linear_fp8(*a, *w, out.half()),
                 lambda: ops.linear_fp8(*a, *w, out.T), lambda: ops.linear_fp8(*a, *w, out[:1].expand(4, 300)), lambda: ops.linear_fp8(*a, w[0].cpu(), w[1], out),
                 lambda: ops.linear_fp8(*a, *w, out.bfloat16(), accumulate=True), lambda: ops.linear_swiglu_fp8(*a, *w, out.bfloat16()),
                 lambda: ops.linear_swiglu_fp8(*a, *weight8(ops, randn(g, 512, 256)), out[:, :256].bfloat16(), act="clamped"),
                 lambda: ops.quantize_fp8(x[:, :255], *a), lambda: ops.quantize_fp8(x.double(), *a), lambda: ops.quantize_fp8(x, a[0], a[1][:2]),
                 lambda: ops.quantize_fp8(x.T, *ops.fp8_rows(256, 4, DEV)), lambda: ops.rms_norm_fp8(x, x[0].cpu(), 1e-5, *a),
                 lambda: ops.rms_norm_fp8(x[:, ::2], x[0, ::2], 1e-5, *ops.fp8_rows(4, 128, DEV)), lambda: ops.quantize_weight_fp8(x, a[0], a[1])):
        before = ops.launches
        with pytest.raises(ops.KernelError):
            call()
        assert ops.launches <= before + 1      # (some prepare an operand with a launch of their own)
    assert bool((out == 7.0).all())


def test_threads_on_streams_of_their_own(ops):
    """Two threads at once, each on a stream of its own, with shared weights: what each gets alone."""
    import threading
    g = rng(5)
    w, gu = weight8(ops, randn(g, 500, 512)), gated_weight(ops, g, 300, 512)
    rows = [rows8(ops, randn(g, m, 512)) for m in (3, 150)]
    want = []
    for a in rows:
        o, h = torch.empty(a[0].shape[0], 500, device=DEV), ops.fp8_rows(a[0].shape[0], 300, DEV)
        ops.linear_fp8(*a, *w, o)
        ops.linear_swiglu_fp8(*a, *gu, *h)
        want.append((o, h[0].float(), h[1].float()))
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                a = rows[i]
                o, h = torch.empty_like(want[i][0]), ops.fp8_rows(a[0].shape[0], 300, DEV)
                for _ in range(200):
                    ops.linear_fp8(*a, *w, o)
                    ops.linear_swiglu_fp8(*a, *gu, *h)
                torch.cuda.current_stream().synchronize()
                got[i] = (o, h[0].float(), h[1].float())
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    assert all(torch.equal(x, y) for p, q in zip(got, want) for x, y in zip(p, q))


# ---------------------------------------------------------------------------------------------- ends of the range


@pytest.mark.parametrize("m,k", [(2, 25601), (3, 25700), (2, 28672), (2, 28800), (1, 32768), (2, 32769), (300, 25700), (300, 28800), (300, 32768)])
def test_normed_rows_of_the_widest_ctas(ops, m, k):
    test_normed_rows(ops, m, k)


@pytest.mark.parametrize("m", [3, 100, 2400])
def test_relu_of_gates_and_ups_at_the_ends(ops, m):
    """Gate sums of 2^-100, 2^-110, 2^100 and -2^100 beside up sums of 1.5 * 2^127, 2^127, 2^-100 and 2^127: the sums are exact, the
    product has one rounding to 32 bits and one to bfloat16, below 2^-126 a multiple of 2^-133."""
    sums, ups = [2.0 ** -100, 2.0 ** -110, 2.0 ** 100, -2.0 ** 100], [1.5 * 2.0 ** 127, -2.0 ** 127, 2.0 ** -100, 2.0 ** 127]
    a = rows8(ops, torch.ones(m, 128, device=DEV))
    w = torch.ones(4, 2, 128, 128, device=DEV)
    for b in range(4):
        w[b, 0], w[b, 1] = math.copysign(1.0, sums[b]), math.copysign(1.0, ups[b])
    w = weight8(ops, w.view(-1, 128))
    for b in range(4):
        w[1][2 * b], w[1][2 * b + 1] = abs(sums[b]) * 2.0 ** -7 * 2.0 ** -8, abs(ups[b]) * 2.0 ** -7 * 2.0 ** -8      # (the values are 256, and 256 * 2^-8)
    want = (torch.tensor(sums, dtype=torch.float64).clamp(min=0) * torch.tensor(ups, dtype=torch.float64)).repeat_interleave(128).to(DEV)
    out = torch.empty(m, 512, dtype=torch.bfloat16, device=DEV)
    ops.linear_swiglu_fp8(*a, *w, out, act="relu")
    assert bool(((out.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -23) * want.abs() + 2.0 ** -133).all())
    ops.check_status()


def exact_gate(g, u, act, limit):
    """The gates in 64 bits with nothing lost far below zero, and the sigmoid's argument."""
    if act == "clamped":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
    t = {"silu": g, "clamped": 1.702 * g, "gelu_tanh": 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)}[act]
    return g * torch.sigmoid(t) * u, t


@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("clamped", 2.0 ** 125), ("gelu_tanh", 0.0)])
@pytest.mark.parametrize("m", [3, 100, 2400])
def test_gates_far_below_zero(ops, m, act, limit):
    """Gate sums whose sigmoid is about to leave 32 bits (arguments of -80 to -110, and sums of -2^135, infinite in 32 bits) and small and
    large positive ones, beside up sums of 2^120 and 1.5 * 2^127.  The argument has three roundings and the constants' (4 * 2^-24 of it), the
    gate 2^-19 of the value; exp is a multiple of 2^-149 there and off by one, times the gate's input."""
    at = {"silu": 1.0, "clamped": 1.702, "gelu_tanh": None}[act]
    args = [80.0, 87.3, 87.4, 87.9, 88.1, 88.6, 89.0, 95.0, 102.0, 110.0]
    if at is None:      # the sum whose argument this is, by Newton's steps
        sums = []
        for t in args:
            x = 10.0
            for _ in range(50):
                x -= (2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3) - t) / (2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x))
            sums.append(-x)
    else:
        sums = [-t / at for t in args]
    sums += [-2.0 ** 135, 2.0 ** -100, 0.5, 3.0]
    ups = [2.0 ** 120] * 10 + [2.0, 1.5 * 2.0 ** 127, 1.5 * 2.0 ** 127, 2.0 ** 100]
    a = rows8(ops, torch.ones(m, 128, device=DEV))
    w = torch.ones(len(sums), 2, 128, 128, device=DEV)
    for b, s in enumerate(sums):
        w[b, 0] = math.copysign(1.0, s)
    w = weight8(ops, w.view(-1, 128))
    for b, (s, u) in enumerate(zip(sums, ups)):
        w[1][2 * b], w[1][2 * b + 1] = abs(s) * 2.0 ** -15, u * 2.0 ** -15      # (the values are 256, and 256 * 2^-8)
    y = fu.product(*a, *w)[0].view(m, -1, 2, 128)
    g, u = (y[:, :, side].reshape(m, -1) for side in (0, 1))
    want, t = exact_gate(g, u, act, limit)
    out = torch.empty(m, 128 * len(sums), dtype=torch.bfloat16, device=DEV)
    ops.linear_swiglu_fp8(*a, *w, out, act=act, limit=limit)
    small = want.abs() < 2.0 ** 127
    assert bool(small[:, : 12 * 128].all())
    off = (2.0 ** -8 + 2.0 ** -18 + 4 * 2.0 ** -24 * t.abs().clamp(max=200)) * want.abs() + \
        (2 * g.abs().clamp(max=200) + 2) * 2.0 ** -149 * (u.clamp(-limit, limit) + 1 if act == "clamped" else u).abs() + 2.0 ** -126
    got = out.double()
    assert not bool(torch.isnan(got).any())
    assert bool(((got - want).abs() <= off)[small].all()) and bool((got[~small].abs() > 2.0 ** 126).all())
    ops.check_status()


def far_scales(g, m, n, k):
    """The first three groups of K.  Rows 0, 4, ...: scale 2^100 on a group whose block has 2^30, with one value of 2^-9 against columns that are
    zero (the first hundred) or hold 2^-9 (2^-18 * 2^130 is a normal float, 2^130 is none); rows 1, 5, ...: 2^-126 on blocks of
    1.3 * 2^-12; rows 2, 6, ...: 2^-127 on blocks of 1.7 * 2^-36 (2^-163, and sums of 2^18); the others: nothing far."""
    a = torch.randn(m, k, generator=g, device=DEV) * 100
    w = torch.randn(n, k, generator=g, device=DEV) * 100
    e = torch.full((m, fu.groups(k)), 127, device=DEV)
    a[:, :128] = 0
    a[0::4, 5] = 2.0 ** -9
    w[:, :128] = 0
    w[100:, :128] = 2.0 ** -9
    e[0::4, 0], e[1::4, 1], e[2::4, 2] = 227, 1, 0
    a[1::4, 256:] = 0
    a[2::4, 128:256] = 0
    a[1::4, 384:], a[2::4, 384:] = 0, 0
    rows = (a.clamp(-448, 448).to(torch.float8_e4m3fn), e.to(torch.uint8).view(torch.float8_e8m0fnu))
    blocks = torch.ones(fu.groups(n), fu.groups(k), device=DEV)
    blocks[:, :3] = torch.tensor([2.0 ** 30, 1.3 * 2.0 ** -12, 1.7 * 2.0 ** -36], device=DEV)
    return rows, w.clamp(-448, 448).to(torch.float8_e4m3fn), blocks


def in_room(ops, rows, weight):
    """The same values in rows that start on 16 bytes."""
    a, w = ops.fp8_rows(*rows[0].shape, DEV), ops.fp8_weight(*weight[0].shape, DEV)
    for room, t in zip(a + w, rows + weight):
        room.copy_(t)
    return a, w


@pytest.mark.parametrize("m,n,k", [(4, 130, 300), (5, 700, 1100), (40, 14336, 300), (64, 40000, 300), (128, 4096, 2304), (600, 3000, 300), (700, 8192, 400)])
def test_scales_whose_product_is_no_normal_float(ops, m, n, k):
    """The row's scale times the block's may be far outside of 32 bits where the result is not; what is left of a sum below 2^-126 is
    a multiple of 2^-149."""
    rows, w, blocks = far_scales(rng(m + n), m, n, k)
    a, w = in_room(ops, rows, (w, blocks))
    want, off = fu.product(*a, *w)
    assert bool((want.abs() < 2.0 ** 120).all())
    out = torch.empty(m, n, device=DEV)
    ops.linear_fp8(*a, *w, out)
    assert bool(((out - want).abs() <= off + 2.0 ** -24 * want.abs() + 3 * 2.0 ** -149).all())
    stream = randn(rng(m), m, n)
    acc = stream.clone()
    ops.linear_fp8(*a, *w, acc, accumulate=True)
    assert bool(((acc - (stream + want)).abs() <= off + 2.0 ** -24 * ((stream + want).abs() + want.abs() + off)).all())
    ops.check_status()


@pytest.mark.parametrize("m,n,k", [(4, 530, 300), (5, 700, 1100), (600, 3000, 300), (700, 8192, 400)])
def test_block_scales_of_zero_below_zero_and_nan(ops, m, n, k):
    """The first block of columns has scales of 0 (a product of 0, and of -0), the second below zero, the third a NaN."""
    g = rng(m + n)
    a, w = rows8(ops, randn(g, m, k)), weight8(ops, randn(g, n, k))
    w[1][0], w[1][1], w[1][2, 1] = 0.0, -w[1][1], math.nan
    w[1][0, 1] = -0.0
    out, stream = torch.empty(m, n, device=DEV), randn(g, m, n)
    acc = stream.clone()
    ops.linear_fp8(*a, *w, out)
    ops.linear_fp8(*a, *w, acc, accumulate=True)
    want, off = fu.product(*a, *w)
    assert bool((out[:, :128] == 0).all()) and bool((acc[:, :128] == stream[:, :128]).all())
    assert bool(torch.isnan(out[:, 256:384]).all()) and bool(torch.isnan(acc[:, 256:384]).all())
    keep = torch.arange(n, device=DEV) // 128 != 2
    assert bool(((out - want).abs() <= off + 2.0 ** -24 * want.abs())[:, keep].all())
    assert bool(((acc - (stream + want)).abs() <= off + 2.0 ** -24 * ((stream + want).abs() + want.abs() + off))[:, keep].all())
    ops.check_status()


@pytest.mark.parametrize("m,i", [(4, 130), (40, 6400), (64, 14336), (700, 2500)])
def test_gated_scales_whose_product_is_no_normal_float(ops, m, i):
    """Rows 0, 2, ...: a group with 2^100 on blocks of 2^30 that hold zeros.  Rows 1, 3, ...: 2^-126 on gate blocks of 1.3 * 2^-24
    (sums of about 2^-133) and up blocks of 2^120.  Gate sums come out as
    multiples of 2^-149, results as multiples of 2^-133."""
    g, k = rng(m + i), 300
    x = torch.randn(m, k, generator=g, device=DEV) * 100
    e = torch.full((m, 3), 127, device=DEV)
    x[:, 256:] = 0
    x[1::2, :128] = 0
    e[0::2, 0], e[1::2, 1] = 227, 1
    b = fu.groups(i)
    w = torch.randn(256 * b, k, generator=g, device=DEV) * 100
    w[:, :128] = 0
    blocks = torch.ones(2 * b, 3, device=DEV)
    blocks[:, 0] = 2.0 ** 30
    blocks[0::2, 1], blocks[1::2, 1] = 1.3 * 2.0 ** -24, 2.0 ** 120
    x[0::2, 128:256] *= 2.0 ** -14
    a, w = in_room(ops, (x.clamp(-448, 448).to(torch.float8_e4m3fn), e.to(torch.uint8).view(torch.float8_e8m0fnu)),
                   (w.clamp(-448, 448).to(torch.float8_e4m3fn), blocks))
    want, off = fu.gated(*a, *w, i, "silu")
    up = fu.product(*a, *w)[0].view(m, -1, 2, 128)[:, :, 1].reshape(m, -1)[:, :i]
    beyond = want.abs() > 2.0 ** 127
    assert not bool(beyond[1::2].any())
    out = torch.empty(m, i, dtype=torch.bfloat16, device=DEV)
    ops.linear_swiglu_fp8(*a, *w, out)
    assert not bool(torch.isnan(out).any())
    assert bool(((out.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off) + 4 * 2.0 ** -149 * (up.abs() + 1) + 2.0 ** -133)[~beyond].all())
    ops.check_status()


@pytest.mark.parametrize("m", [1, 20, 40])
def test_more_than_65535_blocks_of_columns(ops, m):
    g = rng(m)
    n, k = 65536 * 128 + 5, 16
    a, w = rows8(ops, randn(g, m, k)), weight8(ops, randn(g, n, k))
    last = slice(65534 * 128, n)
    out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    ops.linear_fp8(*a, *w, out)
    for part in (slice(0, 300), last):
        scales = w[1][part.start // 128: -(-part.stop // 128)]
        want, off = fu.product(*a, w[0][part], scales)
        assert bool(((out[:, part].double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all())
    ops.check_status()


def test_weights_of_more_than_65535_blocks_of_rows(ops):
    g = rng(1)
    n, k = 65536 * 128 + 5, 16
    x = randn(g, n, k)
    data, scales = weight8(ops, x)
    for part in (slice(0, 300 * 128), slice(65530 * 128, n)):
        want, ws = fu.quantize_weight(x[part])
        assert same(data[part], want) and same(scales[part.start // 128: -(-part.stop // 128)], ws)


@pytest.mark.parametrize("m", [3, 40, 64, 100, 700])
def test_gated_weights_may_be_made_right_before_they_are_read(ops, m):
    g = rng(m)
    i, k = 2500, 1024
    x = [randn(g, 256 * fu.groups(i), k) / math.sqrt(k) for _ in range(4)]
    a, room = rows8(ops, randn(g, m, k)), ops.fp8_weight(256 * fu.groups(i), k, DEV)
    out = [torch.empty(m, i, dtype=torch.bfloat16, device=DEV) for _ in x]
    for w, o in zip(x, out):
        ops.quantize_weight_fp8(w, *room)
        ops.linear_swiglu_fp8(*a, *room, o)
    for w, o in zip(x, out):
        want, off = fu.gated(*a, *weight8(ops, w), i, "silu")
        assert bool(((o.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all())
    ops.check_status()


# ---------------------------------------------------------------------------------------------- which kernel


def kernel_of(m, n, k, gated=False):
    """(which kernel, whether K is cut) of a product of these sizes: 16 to 128 are the rows of A beside a block of columns, 1,128 and 1,256 the
    kernels of large tiles."""
    import ctypes
    from tiny_llm_b200.ops import build
    slices = ctypes.c_int(0)
    kernel = build.load_library("linear_fp8").tllm_linear_fp8_kernel(m, n, k, int(gated), ctypes.byref(slices))
    return kernel, slices.value > 1


@pytest.mark.parametrize("kernel,cut,m,n,k", [
    (16, False, 9, 300, 500), (16, True, 13, 1000, 2100), (16, True, 100, 500, 1100), (32, False, 60, 9000, 400), (32, True, 50, 4100, 4001),
    (64, False, 40, 19000, 129), (64, False, 64, 19001, 1000), (64, True, 50, 2050, 9000), (64, True, 64, 4096, 14336), (128, True, 100, 1300, 7000),
    (128, True, 128, 4100, 2305), (128, True, 200, 2000, 4001), (128, True, 300, 1001, 4000), (1128, False, 300, 4100, 520), (1128, False, 513, 2200, 1001),
    (1128, False, 257, 4300, 129), (1256, False, 1030, 4001, 1000), (1256, False, 2100, 1290, 2000)])
def test_products_of_each_kernel(ops, kernel, cut, m, n, k):
    """What test_products_are_near_64_bits looks at, with the tails of K and of the columns, rows that do not start on 16 bytes and every kind of
    output, on the kernel that is named."""
    assert kernel_of(m, n, k) == (kernel, cut)
    test_products_are_near_64_bits(ops, m, n, k)


@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("clamped", 1.5)])
@pytest.mark.parametrize("kernel,cut,m,i,k", [
    (16, False, 12, 300, 500), (16, True, 8, 1000, 2048), (16, True, 16, 1000, 2100), (16, True, 3, 5632, 2048), (32, False, 40, 6400, 300), (32, True, 64, 2000, 3001),
    (64, False, 64, 10001, 300), (64, True, 64, 1500, 7000), (64, False, 200, 4000, 700), (64, True, 100, 1000, 9001),
    (1256, False, 700, 2501, 650), (1256, False, 1300, 1290, 1111), (1256, False, 513, 5632, 2048)])
def test_gated_products_of_each_kernel(ops, kernel, cut, m, i, k, act, limit):
    assert kernel_of(m, i, k, gated=True) == (kernel, cut)
    test_gated_products(ops, m, i, k, act, limit)


def test_the_kernels_of_the_other_tests(ops):
    """The sizes by which the tests above mean a kernel."""
    assert [kernel_of(m, n, k)[0] for m, n, k in [(4, 130, 300), (5, 700, 1100), (40, 14336, 300), (64, 40000, 300), (128, 4096, 2304), (600, 3000, 300), (700, 8192, 400)]] == \
        [16, 16, 32, 64, 128, 1128, 1256]
    assert [kernel_of(m, i, 300, gated=True)[0] for m, i in [(4, 130), (40, 6400), (64, 14336), (700, 2500)]] == [16, 32, 64, 1256]
    assert [kernel_of(m, 1792, 128, gated=True)[0] for m in (3, 100, 2400)] == [16, 16, 1256]


def test_slices_of_one_round(ops):
    """K is cut so that the tiles still run at once: no more CTAs than two per SM, and fewer slices the more tiles there are."""
    import ctypes
    from tiny_llm_b200.ops import build
    lib, slices = build.load_library("linear_fp8"), ctypes.c_int(0)

    def cut(m, n, k):
        lib.tllm_linear_fp8_kernel(m, n, k, 0, ctypes.byref(slices))
        return slices.value
    places = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    assert cut(8, 2560, 2048) == 4 and cut(8, 128, 128) == 1 and cut(8, 128, 1 << 16) == 8
    for k in (1 << 16, 9216, 2048):
        by_tiles = [cut(8, 128 * tiles, k) for tiles in range(1, 400)]
        assert by_tiles == sorted(by_tiles, reverse=True) and by_tiles[0] == min(8, k // 512) and by_tiles[-1] == 1
        assert all(s * tiles <= places for tiles, s in enumerate(by_tiles, 1) if s > 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(300, 14336), (4000, 1030), (1481, 2550), (1400, 1000), (1200, 4096)])
def test_rows_of_long_runs(ops, m, k, dtype):
    """More groups than the kernel of short runs takes (12,432 of float32, 29,600 of bfloat16), and next to them."""
    test_rows_are_the_nearest_8_bit_values(ops, m, k, dtype)


@pytest.mark.parametrize("m,k", [(3700, 520), (2368, 1000), (2367, 1030), (1184, 2048), (1200, 2050), (600, 4096), (640, 4101), (297, 8192), (330, 8000), (9, 9000), (200, 14336)])
def test_normed_rows_of_few_and_many_groups(ops, m, k):
    """Next to 18,944 groups in all, where a warp gets eight of them instead of one, two or four, and rows of more than 64 groups."""
    test_normed_rows(ops, m, k)


def test_the_first_calls_of_a_process_may_be_captured():
    """Loading, limits and what the runtime is asked happen inside the capture then."""
    import os
    import subprocess
    import sys
    script = """
import torch
from tiny_llm_b200 import ops
g = torch.Generator(device="cuda").manual_seed(0)
x, w = (torch.randn(*s, generator=g, device="cuda") for s in ((700, 640), (4096, 640)))
norm, out, few = torch.ones(640, device="cuda"), torch.zeros(700, 4096, device="cuda"), torch.zeros(3, 4096, device="cuda")
a, b, q, h = ops.fp8_rows(700, 640, "cuda"), ops.fp8_rows(700, 640, "cuda"), ops.fp8_weight(4096, 640, "cuda"), ops.fp8_rows(700, 2048, "cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.quantize_weight_fp8(w, *q)
    ops.rms_norm_fp8(x, norm, 1e-5, *b)
    ops.quantize_fp8(x, *a)
    ops.linear_swiglu_fp8(*b, *q, *h)
    ops.linear_fp8(*a, *q, out)
    ops.linear_fp8(a[0][:3], a[1][:3], *q, few)
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (out, few, h[0].float(), h[1].float())]
ops.linear_fp8(*a, *q, out)
ops.linear_fp8(a[0][:3], a[1][:3], *q, few)
ops.linear_swiglu_fp8(*b, *q, *h)
assert all(torch.equal(x, y) for x, y in zip(got, (out, few, h[0].float(), h[1].float()))) and float(out.norm()) > 0 and float(few.norm()) > 0
ops.check_status()
print("the same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 0 and r.stdout.split("\n")[-2] == "the same", r.stderr
