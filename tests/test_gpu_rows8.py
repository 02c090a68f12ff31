"""Rows of 8-bit numbers on the GPU, operator by operator against plain 64-bit restatements (rows8_util)."""
import math

import pytest
import torch

import mistral_inference_b200 as mi
from mistral_inference_b200.rows8 import Rows8

from . import rows8_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def normal(shape, seed, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=torch.Generator(device=DEV).manual_seed(seed))


def uneven(T, K, seed, dtype):
    """Rows whose entries span many powers of two, zeros among them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = normal((T, K), seed) * torch.exp2(torch.randint(-9, 10, (T, K), device=DEV, generator=g).float())
    x[torch.rand((T, K), device=DEV, generator=g) < 0.1] = 0
    return x.to(dtype)


def assert_same_rows(got: Rows8, x: torch.Tensor):
    codes, scales = U.quantised(x)
    assert torch.equal(got.scales.view(torch.uint8), scales)
    same = got.codes.view(torch.uint8) == codes.view(torch.uint8)
    assert (same | (got.codes.float().isnan() & codes.float().isnan())).all()


# ------------------------------------------------------------------------------------------------------------ quantise
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 4096), (2, 15), (3, 16), (5, 127), (129, 128), (128, 129), (31, 500), (33, 512), (1000, 513), (260, 1003), (7, 5120), (4, 14336)])
def test_quantise(T, K, dtype):
    assert_same_rows(mi.quantise_rows(uneven(T, K, 7 * T + K, dtype)), uneven(T, K, 7 * T + K, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_at_the_borders(dtype):
    """Largest magnitudes next to 448 times a power, zeros of both signs, the smallest and largest numbers, numbers half way between codes."""
    rows = []
    for top in (448.0, 450.0, 446.0, 896.0, 1.75, 1.0, 3.5, 2.0 ** -120, 2.0 ** -133, 3.3e38, 2.0 ** -100 * 448, 2.0 ** -101 * 448):
        row = torch.zeros(256)
        row[0] = -top
        row[1:100] = torch.linspace(-1, 1, 99) * top / 64
        row[130], row[131] = -0.0, top / 7
        rows.append(row)
    half = torch.zeros(256)
    half[:128] = torch.arange(128) * 0.25  # (448 as the largest: steps of 0.25 fall half way between codes from 4 on)
    half[0] = 448
    rows.append(half)
    x = torch.stack(rows).to(DEV).to(dtype)
    assert_same_rows(mi.quantise_rows(x), x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_blocks_that_hold_no_number(dtype, bad):
    x = uneven(40, 700, 3, dtype)
    for r, k in [(0, 0), (3, 127), (3, 128), (20, 699), (39, 512)]:
        x[r, k] = bad
    got = mi.quantise_rows(x)
    assert_same_rows(got, x)
    nan = got.numbers().isnan()
    assert nan[0, :128].all() and not nan[0, 128:].any() and nan[3, :256].all() and not nan[3, 256:].any() and nan[20, 640:].all() and not nan[1].any()


@pytest.mark.parametrize("offset,ld", [(0, 640), (8, 640), (1, 640), (0, 643), (4, 644)])
def test_rows_of_wider_matrices(offset, ld):
    for dtype in (torch.bfloat16, torch.float32):
        wide = uneven(50, ld, 11, dtype)
        x = wide[:, offset: offset + 600]
        assert_same_rows(mi.quantise_rows(x), x)


def test_numbers_and_exponents():
    x = uneven(200, 900, 5, torch.float32)
    got = mi.quantise_rows(x)
    assert torch.equal(got.numbers(torch.float64), U.numbers(got.codes, got.scales, 900))
    assert torch.equal(got.numbers(torch.bfloat16).double(), got.numbers(torch.float64))  # four bits and a power: exact in 16 bits
    assert torch.equal(got.exponents().long(), U.exponent(U.blocks_of(x).abs().amax(2)))


# ---------------------------------------------------------------------------------------------------------------- norm
def norm_in_64_bits(x, w, eps, add):
    h = x if add is None else (x.double() + add.double()).to(x.dtype)  # (a sum of two 16-bit numbers has one rounding either way)
    y = h.double() / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + eps) * w.double()
    return h, y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_add", [False, True])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 4096), (2, 100), (3, 16), (130, 129), (5, 1003), (32, 5120), (300, 6144), (3, 16385), (2, 40000), (1, 65536)])
def test_norm(T, K, with_add, dtype):
    x, w = normal((T, K), K, 1.3, dtype), (1 + normal((K,), K + 1, 0.2)).to(dtype)
    add = normal((T, K), K + 2, 0.7, dtype) if with_add else None
    rows, h = mi.norm_rows(x, w, 1e-5, add=add)
    want, y = norm_in_64_bits(x, w, 1e-5, add)
    if dtype is torch.bfloat16 or not with_add:
        assert torch.equal(h, want)
    else:
        want, y = norm_in_64_bits(h, w, 1e-5, None)
        assert torch.equal(h, x + add)
    assert (h is x) == (not with_add)
    # K products and additions in 32 bits (at most K / 32 one after another, then a tree), a division, a root, two products: each off by 2^-24 of it, the root halves
    assert_off = y.abs() * (K / 32 + 16) * 2.0 ** -24
    U.assert_rows_near(rows.codes, rows.scales, y, assert_off)


def test_norm_of_zeros_and_of_no_numbers():
    x, w = normal((6, 600), 1, 1.0, torch.bfloat16), torch.ones(600, dtype=torch.bfloat16, device=DEV)
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 599] = math.inf
    rows, _ = mi.norm_rows(x, w, 1e-5)
    assert (rows.numbers()[1] == 0).all() and rows.numbers()[2].isnan().all()
    y = rows.numbers()[3]
    assert y[512:].isnan().all() and (y[:512] == 0).all()  # x / infinity, and infinity / infinity in the last block
    U.assert_rows_near(rows.codes[4:], mi.norm_rows(x[4:], w, 1e-5)[0].scales, norm_in_64_bits(x[4:], w, 1e-5, None)[1], 1e-5)


def test_norm_of_rows_of_wider_matrices():
    for dtype in (torch.bfloat16, torch.float32):
        for off, ld in [(0, 1000), (8, 1000), (3, 1000), (0, 999)]:
            x, add = normal((9, ld), 1, 1.0, dtype)[:, off: off + 900], normal((9, ld), 2, 1.0, dtype)[:, off: off + 900]
            w = normal((1000,), 3, 1.0, dtype)[off: off + 900]
            a, h = mi.norm_rows(x, w, 1e-5, add=add)
            b, g = mi.norm_rows(x.contiguous(), w.clone(), 1e-5, add=add.contiguous())
            assert torch.equal(h, g) and torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))


# ------------------------------------------------------------------------------------------------------------ products
def random_rows(T, K, seed, std=1.0):
    return mi.quantise_rows(normal((T, K), seed, std) * torch.exp2(torch.randint(-3, 4, (T, -(-K // 128)), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))
                                                                   .float()).repeat_interleave(128, 1)[:, :K])


SIZES = [(1, 128, 128), (1, 1, 1), (1, 6144, 4096), (2, 130, 200), (5, 1000, 513), (16, 300, 1003), (17, 256, 640), (32, 5120, 1024), (33, 257, 2000), (64, 4096, 4096), (100, 700, 900),
         (128, 512, 512), (129, 1001, 1152), (200, 2048, 128), (256, 256, 4096), (300, 4099, 700), (513, 1536, 2048), (777, 6144, 512), (1102, 2048, 1000), (777, 6144, 4096), (129, 4096, 14336), (1500, 5000, 2700)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,N,K", SIZES)
def test_multiply(T, N, K, dtype):
    x, w = random_rows(T, K, T + K), random_rows(N, K, N + K, 0.1)
    y, off = U.product(U.numbers(x.codes, x.scales, K), U.numbers(w.codes, w.scales, K))
    got = mi.multiply_rows(x, w, dtype=dtype)
    assert got.dtype is dtype and got.shape == (T, N)
    if dtype is torch.bfloat16:
        off = off + (y.abs() + off) * 2.0 ** -8
    bad = (got.double() - y).abs() > off
    assert not bad.any(), f"{int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {y[bad][0]}"


@pytest.mark.parametrize("T,H,K", [(1, 128, 128), (1, 1, 1), (1, 14336, 4096), (3, 100, 200), (16, 700, 513), (32, 1003, 1003), (48, 640, 5120), (64, 2048, 640), (65, 64, 900), (128, 384, 512),
                                   (129, 500, 1152), (256, 128, 4096), (300, 2050, 700), (1102, 1024, 1000), (777, 3001, 4096), (140, 14336, 2560)])
def test_gate(T, H, K):
    x, w = random_rows(T, K, T + K), random_rows(2 * H, K, H + K, 1.5 * K ** -0.5)
    y, off = U.product(U.numbers(x.codes, x.scales, K), U.numbers(w.codes, w.scales, K))
    gate, up = y[:, 0::2], y[:, 1::2]
    g = gate * torch.sigmoid(gate) * up
    # silu's slope is within [-0.1, 1.1]; e^-x is 2^(-x log2 e) of a product that is off by 2^-24 of its magnitude: up to |x| 2^-24, beside a few units of 2^-22 in all
    far = 1.1 * off[:, 0::2] * (up.abs() + off[:, 1::2]) + gate.abs() * off[:, 1::2] + g.abs() * (8 + gate.abs() / 2) * 2.0 ** -22
    rows = mi.gate_rows(x, w)
    assert rows.cols == H and rows.rows == T
    U.assert_rows_near(rows.codes, rows.scales, g, far)


@pytest.mark.parametrize("T,N,K", [(33, 4096, 1024), (65, 4096, 2048), (100, 2048, 1900), (128, 5120, 2560), (96, 8192, 1024), (48, 2560, 4096), (16, 2048, 4096), (40, 16384, 512)])
def test_splits_of_few_tokens(T, N, K):
    """The sizes at which a product for a few tokens changes how many CTAs take its features, and how many of them an SM holds; the same bits each time."""
    x, w = random_rows(T, K, T + K), random_rows(N, K, N + K, 1.5 * K ** -0.5)
    y, off = U.product(U.numbers(x.codes, x.scales, K), U.numbers(w.codes, w.scales, K))
    got = mi.multiply_rows(x, w, dtype=torch.float32)
    assert ((got.double() - y).abs() <= off).all()
    gate, up = y[:, 0::2], y[:, 1::2]
    g = gate * torch.sigmoid(gate) * up
    far = 1.1 * off[:, 0::2] * (up.abs() + off[:, 1::2]) + gate.abs() * off[:, 1::2] + g.abs() * (8 + gate.abs() / 2) * 2.0 ** -22
    rows = mi.gate_rows(x, w)
    U.assert_rows_near(rows.codes, rows.scales, g, far)
    for _ in range(3):
        assert torch.equal(mi.multiply_rows(x, w, dtype=torch.float32), got)
        again = mi.gate_rows(x, w)
        assert torch.equal(again.codes, rows.codes) and torch.equal(again.scales, rows.scales)


def test_many_clusters_of_little_shared_memory():
    """Each token column takes two columns of tensor memory, of which an SM has 512: more CTAs than that come one after another, whatever their shared memory, on one stream and on four."""
    streams = [torch.cuda.Stream() for _ in range(4)]
    for T, N, K in ((128, 40000, 128), (128, 4096, 1024), (64, 40000, 128), (100, 4096, 512)):
        x, w = random_rows(T, K, T + K), random_rows(N, K, N + K, 1.5 * K ** -0.5)
        want, units = mi.multiply_rows(x, w), mi.gate_rows(x, w)
        torch.cuda.synchronize()
        got = []
        for i in range(24):
            with torch.cuda.stream(streams[i % 4]):
                got.append(mi.multiply_rows(x, w) if i % 3 == 0 else mi.gate_rows(x, w))
        torch.cuda.synchronize()
        for i, g in enumerate(got):
            if i % 3 == 0:
                assert torch.equal(g, want), (T, N, K, i)
            else:
                assert torch.equal(g.codes, units.codes) and torch.equal(g.scales, units.scales), (T, N, K, i)


def test_scales_of_every_row_and_block_reach_their_products():
    """One entry a block: every power is seen by itself."""
    for T, N in ((4, 260), (40, 130), (300, 260)):
        K = 128 * 9
        x, w = torch.zeros(T, K, device=DEV), torch.zeros(N, K, device=DEV)
        for b in range(9):
            x[:, 128 * b + 5 * b] = torch.exp2((torch.arange(T, device=DEV) * 7 + b * 3) % 23 - 11.0)
        for b in range(9):
            one = torch.zeros_like(w)
            one[:, 128 * b + 5 * b] = torch.exp2((torch.arange(N, device=DEV) * 5 + b) % 19 - 9.0)
            got = mi.multiply_rows(mi.quantise_rows(x), mi.quantise_rows(one), dtype=torch.float32)
            assert torch.equal(got, x[:, 128 * b + 5 * b, None] * one[None, :, 128 * b + 5 * b]), (T, N, b)


def test_a_row_of_no_numbers_stays_alone():
    for T in (3, 40, 200):
        x, w = normal((T, 700), 1), normal((300, 700), 2)
        x[1, 600] = math.nan
        w[7, 3] = math.inf
        y = mi.multiply_rows(mi.quantise_rows(x), mi.quantise_rows(w))
        nan = y.isnan()
        assert nan[1].all() and nan[:, 7].all()
        nan[1] = False
        nan[:, 7] = False
        assert not nan.any()
        g = mi.gate_rows(mi.quantise_rows(x), mi.quantise_rows(w)).numbers().isnan()
        assert g[1].all() and g[:, :128].all()  # feature 7 is unit 3: its block of each row
        g[1] = False
        assert not g[:, 128:].any()


def test_out_may_be_part_of_wider_rows():
    for T in (2, 60, 300):
        x, w = random_rows(T, 640, 1), random_rows(500, 640, 2)
        for dtype in (torch.bfloat16, torch.float32):
            want = mi.multiply_rows(x, w, dtype=dtype)
            for off, ld in [(0, 512), (8, 512), (3, 517)]:
                wide = torch.full((T, ld), 7.0, dtype=dtype, device=DEV)
                part = wide[:, off: off + 500]
                assert mi.multiply_rows(x, w, out=part) is part and torch.equal(part, want)
                assert (wide[:, :off] == 7).all() and (wide[:, off + 500:] == 7).all()


def test_no_rows():
    x = torch.empty(0, 300, dtype=torch.bfloat16, device=DEV)
    rows = mi.quantise_rows(x)
    normed, h = mi.norm_rows(x, torch.ones(300, dtype=torch.bfloat16, device=DEV), 1e-5, add=x)
    w = random_rows(100, 300, 1)
    assert rows.rows == normed.rows == 0 and h.shape == (0, 300) and mi.multiply_rows(rows, w).shape == (0, 100) and mi.gate_rows(rows, w).rows == 0


# ------------------------------------------------------------------------------------------------------------ how calls are made
def same(a, b):
    if isinstance(a, Rows8):
        return torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))
    return torch.equal(a, b)


def chain(x, weight, wqkv, w13, w2):
    """A sublayer and the next as a layer runs them."""
    rows, h = mi.norm_rows(x, weight, 1e-5)
    a = mi.multiply_rows(rows, wqkv)
    rows, h = mi.norm_rows(h, weight, 1e-5, add=a[:, : x.shape[1]])
    g = mi.gate_rows(rows, w13)
    return h, mi.multiply_rows(mi.quantise_rows(a), wqkv, dtype=torch.float32), g, mi.multiply_rows(g, w2)


def chain_inputs(T, K, H, seed):
    return (normal((T, K), seed, 1.0, torch.bfloat16), (1 + normal((K,), seed + 1, 0.1)).to(torch.bfloat16), random_rows(K, K, seed + 2, K ** -0.5), random_rows(2 * H, K, seed + 3, K ** -0.5),
            random_rows(K, H, seed + 4, H ** -0.5))


@pytest.mark.parametrize("T", [1, 20, 128, 129, 600])
def test_a_run_of_them_against_64_bits(T):
    """Each operator on what the one before it gave: rounded where that is rounded, by the bounds of each."""
    K, H = 640, 1100
    x, weight, wqkv, w13, w2 = chain_inputs(T, K, H, 3 * T)
    h, again, g, y = chain(x, weight, wqkv, w13, w2)
    rows, _ = mi.norm_rows(x, weight, 1e-5)
    want, off = U.product(U.numbers(rows.codes, rows.scales, K), U.numbers(wqkv.codes, wqkv.scales, K))
    a = mi.multiply_rows(rows, wqkv)
    assert ((a.double() - want).abs() <= off + (want.abs() + off) * 2.0 ** -8).all() and torch.equal(h, x + a)
    want, off = U.product(U.numbers(g.codes, g.scales, H), U.numbers(w2.codes, w2.scales, H))
    assert ((y.double() - want).abs() <= off + (want.abs() + off) * 2.0 ** -8).all()
    # and the whole against 64 bits without any rounding in between: four roundings to 8 bits (2^-4 at most, some 2^-5.3 on average, of either sign) of each product's terms
    n = lambda t: t.double() / torch.sqrt((t.double() ** 2).mean(1, keepdim=True) + 1e-5) * weight.double()  # noqa: E731
    e = n(x) @ U.numbers(wqkv.codes, wqkv.scales, K).t()
    z = n(x.double() + e) @ U.numbers(w13.codes, w13.scales, K).t()
    z = (z[:, 0::2] * torch.sigmoid(z[:, 0::2]) * z[:, 1::2]) @ U.numbers(w2.codes, w2.scales, H).t()
    assert (y.double() - z).norm() <= 2.0 ** -3 * z.norm()
    assert again.isfinite().all()


@pytest.mark.parametrize("T", [1, 40, 129, 300])
def test_every_call_gives_the_same_bits(T):
    args = chain_inputs(T, 1000, 1300, T)
    first = chain(*args)
    for _ in range(20):
        assert all(same(a, b) for a, b in zip(first, chain(*args)))


@pytest.mark.parametrize("T", [3, 200])
def test_captured_graphs_on_two_streams_at_once(T):
    """Two graphs of the same calls share weights and nothing else: replayed at the same time, each has its own results."""
    x, weight, *ws = chain_inputs(T, 2048, 2304, T)
    torch.cuda.synchronize()
    for w in ws:
        w.fixed = True
    ins, outs, graphs, want = [], [], [], []
    for i in range(2):
        ins.append(normal((T, 2048), 50 + i, 1.0, torch.bfloat16))
        want.append(chain(ins[i], weight, *ws))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(chain(ins[i], weight, *ws))
        graphs.append((g, s))
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same(a, b) for a, b in zip(outs[i], want[i]))


def test_two_threads_at_once():
    """Each on a stream of its own: the calls let go of the interpreter while they launch."""
    import threading
    args = [chain_inputs(t, 1000, 1200, t) for t in (5, 300)]
    want = [chain(*a) for a in args]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = chain(*args[i])
                torch.cuda.current_stream().synchronize()
                if not all(same(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_weights_written_just_before():
    """Weights that are not fixed are read behind what writes them, whatever runs in between."""
    for T in (2, 60, 200):
        x = random_rows(T, 4096, 1)
        big = normal((6144, 4096), 2)
        want = mi.multiply_rows(x, mi.quantise_rows(big * 2))
        torch.cuda.synchronize()
        for _ in range(10):
            junk = mi.quantise_rows(big)
            w = mi.quantise_rows(big * 2)
            got = mi.multiply_rows(x, w)
            del junk, w
            assert torch.equal(got, want)


def test_rows_cut_between_tiles():
    """Rows from a multiple of 128 on are a matrix of their own: no copy is needed."""
    x, w = random_rows(700, 900, 1), random_rows(300, 900, 2)
    part, head = Rows8(x.codes[256:], x.scales[2:], 900), Rows8(x.codes[:256], x.scales[:2], 900)
    assert torch.equal(part.numbers(), x.numbers()[256:]) and torch.equal(head.numbers(), x.numbers()[:256])
    for a, b in ((part, w), (w, head), (head, part)):
        y, off = U.product(a.numbers(torch.float64), b.numbers(torch.float64))
        assert ((mi.multiply_rows(a, b, dtype=torch.float32).double() - y).abs() <= off).all()


def test_scales_that_are_no_numbers_and_the_smallest():
    for T in (4, 200):
        x, w = random_rows(T, 512, 1), random_rows(140, 512, 2)
        x.scales.view(torch.uint8)[0, 0, 2, 0, 1] = 255  # row 2, block 1
        y = mi.multiply_rows(x, w, dtype=torch.float32)
        nan = y.isnan()
        assert nan[2].all() and not nan[:2].any() and not nan[3:].any()
        w.scales.view(torch.uint8)[0, 0, 5, 0, :] = 0     # 2^-127: its products with powers near 1 are 0 or next to it
        assert (mi.multiply_rows(x, w, dtype=torch.float32)[3:, 5].abs() <= 2.0 ** -90).all()


def test_tensors_of_another_stream():
    x, weight, *ws = chain_inputs(30, 640, 700, 9)
    want = chain(x, weight, *ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(x, weight, *ws)
    torch.cuda.current_stream().wait_stream(side)
    assert all(same(a, b) for a, b in zip(got, want))


def test_results_behind_32_bit_offsets():
    """More than 2^31 numbers: the last rows are where they belong."""
    T, N, K = 70000, 32768, 128
    x, w = random_rows(T, K, 1), random_rows(N, K, 2)
    wv = U.numbers(w.codes, w.scales, K)
    y = mi.multiply_rows(x, w)
    assert y.numel() > 2 ** 31
    for r0 in (0, 65500, T - 100):
        want, off = U.product(x.numbers(torch.float64)[r0: r0 + 100], wv)
        assert ((y[r0: r0 + 100].double() - want).abs() <= off + (want.abs() + off) * 2.0 ** -8).all()
    rows = mi.quantise_rows(y)
    tail = mi.quantise_rows(y[69888:])  # (from a whole tile on)
    assert torch.equal(rows.codes[69888:].view(torch.uint8), tail.codes.view(torch.uint8)) and torch.equal(rows.scales[546:].view(torch.uint8), tail.scales.view(torch.uint8))
    weight = torch.ones(N, dtype=torch.bfloat16, device=DEV)
    normed, h = mi.norm_rows(y, weight, 1e-5, add=y)
    assert torch.equal(h[-50:], y[-50:] + y[-50:])
    tail, _ = mi.norm_rows(y[69888:], weight, 1e-5, add=y[69888:])
    assert torch.equal(normed.codes[69888:].view(torch.uint8), tail.codes.view(torch.uint8)) and torch.equal(normed.scales[546:].view(torch.uint8), tail.scales.view(torch.uint8))
    del y, rows, normed, h
    wide = mi.gate_rows(x, random_rows(2 * N, K, 3))
    part = mi.gate_rows(Rows8(x.codes[69888:], x.scales[546:], K), random_rows(2 * N, K, 3))
    assert wide.codes.numel() > 2 ** 31 and torch.equal(wide.scales[546:].view(torch.uint8), part.scales.view(torch.uint8)) and torch.equal(wide.codes[69888:].view(torch.uint8), part.codes.view(torch.uint8))


def test_results_of_empty_and_refused_calls():
    x, w = random_rows(3, 200, 1), random_rows(4, 200, 2)
    bf = torch.bfloat16
    for call in (lambda: mi.multiply_rows(x, random_rows(4, 201, 1)), lambda: mi.multiply_rows(x, w, dtype=torch.float16), lambda: mi.gate_rows(x, random_rows(3, 200, 1)),
                 lambda: mi.multiply_rows(x, w, out=torch.empty(3, 5, device=DEV, dtype=bf)), lambda: mi.multiply_rows(x, w, out=torch.empty(4, 3, device=DEV, dtype=bf).t()),
                 lambda: mi.multiply_rows(x, Rows8(w.codes, w.scales, 100)), lambda: mi.multiply_rows(Rows8(x.codes.view(torch.uint8), x.scales, 200), w),
                 lambda: mi.multiply_rows(Rows8(x.codes, x.scales.cpu(), 200), w), lambda: mi.multiply_rows(Rows8(x.codes[:, :128], x.scales, 100), w),
                 lambda: mi.norm_rows(normal((2, 70000), 1, 1.0, bf), normal((70000,), 1, 1.0, bf), 1e-5), lambda: mi.norm_rows(normal((2, 70), 1, 1.0, bf), normal((70,), 1), 1e-5),
                 lambda: mi.norm_rows(normal((2, 70), 1), normal((70,), 1), 1e-5, add=normal((2, 71), 1)), lambda: mi.quantise_rows(normal((2, 70), 1).half())):
        with pytest.raises(AssertionError):
            call()


def test_results_take_the_type_of_out():
    x, w = random_rows(5, 300, 1), random_rows(40, 300, 2)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.empty(5, 40, dtype=dtype, device=DEV)
        for said in (None, dtype):
            assert mi.multiply_rows(x, w, dtype=said, out=out) is out and torch.equal(out, mi.multiply_rows(x, w, dtype=dtype))
    assert mi.multiply_rows(x, w).dtype is torch.bfloat16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K,offset,ld", [(16400, 1003, 0, 1003), (7000, 2561, 0, 2561), (7000, 2561, 1, 2600), (8200, 2049, 0, 2056), (8200, 2049, 3, 2056), (4096, 4096, 0, 4096), (4100, 4000, 4, 4008), (33000, 17, 5, 31)])
def test_quantise_of_many_rows(T, K, offset, ld, dtype):
    """From 32768 steps of 512 entries on a warp takes four of them: rows whose steps are no multiple of four, that begin anywhere, and blocks that hold no number, bit for bit."""
    assert T * -(-K // 512) >= 32768
    x = uneven(T, ld, T + K, dtype)[:, offset: offset + K]
    for r, k in [(0, K - 1), (T - 1, 0), (T // 2, K // 2), (T - 130, min(K - 1, 511))]:
        x[r, k] = math.nan if r % 2 else math.inf
    assert_same_rows(mi.quantise_rows(x), x)


@pytest.mark.parametrize("T", [100, 250])
def test_gates_far_from_zero(T):
    """Units of exact gates from -104 to 104 and ups up to 2^60, each in a block of its own.  Off by (3 + |gate| / 3) 2^-22 of themselves, and below -87, where silu ends, by 2^-119 of the up."""
    gates = torch.tensor([s * m * 2.0 ** e for e in range(-2, 6) for m in (1.0, 1.125, 1.375, 1.625, 1.75) for s in (-1, 1)] + [s * v for v in (72.0, 80.0, 88.0, 96.0, 104.0) for s in (-1, 1)], device=DEV)
    x = torch.zeros(T, 256, device=DEV)
    i = torch.arange(T, device=DEV)
    x[:, 0] = gates[i * 7 % len(gates)]
    x[:, 128] = torch.exp2((i * 11 % 61).float()) * torch.where(i % 2 == 0, 1.0, -1.0)
    w = torch.zeros(2, 256, device=DEV)
    w[0, 0] = w[1, 128] = 1
    a = mi.quantise_rows(x)
    assert torch.equal(a.numbers(), x)
    rows = mi.gate_rows(a, mi.quantise_rows(w))
    gate, up = x[:, :1].double(), x[:, 128:129].double()
    y = gate * torch.sigmoid(gate) * up
    U.assert_rows_near(rows.codes, rows.scales, y, y.abs() * (3 + gate.abs() / 3) * 2.0 ** -22 + torch.where(gate < -87, 2.0 ** -119, 0.0) * up.abs())


MOST = 1 << 24


def test_as_many_rows_as_there_may_be():
    """2^24 rows of one entry: every row's code and power, and its products with three features, which are exact."""
    i = torch.arange(MOST, device=DEV)
    x = ((1 + i % 8 / 8) * torch.exp2((i // 8 % 20 - 9).float())).to(torch.bfloat16)[:, None]
    rows = mi.quantise_rows(x)
    assert torch.equal(rows.codes[:, 0].float() * torch.exp2(rows.exponents()[:, 0].float()), x[:, 0].float())
    assert int(rows.codes.view(torch.int32)[:, 1:].count_nonzero()) == 0  # (the first four codes of a row are one word)
    w = mi.quantise_rows(torch.tensor([[1.5], [-1.0], [0.25]], device=DEV))
    y = mi.multiply_rows(rows, w, dtype=torch.float32)
    assert torch.equal(y, x.float() * torch.tensor([1.5, -1.0, 0.25], device=DEV))
    del y
    one = mi.quantise_rows(torch.ones(1, 1, device=DEV))
    assert torch.equal(mi.multiply_rows(one, rows, dtype=torch.float32)[0], x[:, 0].float())
    units = mi.gate_rows(one, rows)
    gate, up = x[0::2, 0].double()[None], x[1::2, 0].double()[None]
    y = gate * torch.sigmoid(gate) * up
    U.assert_rows_near(units.codes, units.scales, y, y.abs() * (3 + gate.abs() / 3) * 2.0 ** -22)


@pytest.mark.parametrize("T", [2, 130])
def test_rows_as_long_as_they_may_be(T):
    """2^24 entries, a few of which are not zero: sums that are exact."""
    at = [0, 127, 5_000_000, (1 << 23) + 5, MOST - 129, MOST - 1]
    x, w = torch.zeros(T, MOST, dtype=torch.bfloat16, device=DEV), torch.zeros(3, MOST, dtype=torch.bfloat16, device=DEV)
    for j, k in enumerate(at):
        x[:, k] = (torch.arange(T, device=DEV) * 5 + j * 3) % 15 + 1
        w[:, k] = torch.tensor([1.0, -2.0, 0.5], device=DEV) * (j + 1)
    y = x[:, at].float() @ w[:, at].float().t()
    x = mi.quantise_rows(x)
    w = mi.quantise_rows(w)
    for k in at:
        assert torch.equal(x.exponents()[:, k // 128] > -100, torch.ones(T, dtype=torch.bool, device=DEV))
    got = mi.multiply_rows(x, w, dtype=torch.float32)
    assert torch.equal(got, y)
