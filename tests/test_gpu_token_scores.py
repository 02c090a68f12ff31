"""Scores of tokens on the GPU against 64 bits."""
import math

import pytest
import torch

import mistral_inference_b200 as mi

from . import paged_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def logits_of(T, V, seed, std=3.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, V, generator=g) * std).to(torch.bfloat16).to(dtype)  # equal values are common


def check(x, targets, top):
    s = mi.token_scores(x.to(DEV), None if targets is None else targets.to(DEV), top=top)
    lp, ent, ids, lps = U.scores_ref(x, targets, top)
    assert s.top_ids.cpu().tolist() == ids.tolist()
    # x - m and its exponential in fp32: 2^-24 of the exponent and 2 ulp (2^-22) each, exponents up to 2^7 of those that count; sums of positive numbers by threads and in trees, at most
    # 2^5 steps of 2^-24 each: 2^-17 of the sum, absolute in its logarithm; the difference with the target's logit rounds once (2^-24 of up to 2^8).  Entropies: the same of both sums.
    for got, want in ((s.logprob, lp), (s.entropy, ent), (s.top_logprobs, lps)):
        if want is None:
            assert got is None
            continue
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan())
        fin = want.isfinite()
        assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
        assert ((got - want).abs()[fin] <= 2.0 ** -17 + 2.0 ** -15 * want.abs()[fin].clamp(max=16)).all(), (got - want).abs()[fin].max()
    return s


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1003, 8192, 8193, 32000, 131072, 200001])
@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores(V, T, dtype):
    x = logits_of(T, V, V, dtype=dtype)
    targets = torch.tensor([(7919 * i) % V if i % 3 != 1 else -1 for i in range(T)])
    for top in sorted({0, 1, min(V, 5), min(V, 64)}):
        check(x, targets, top)
    check(x, None, min(V, 3))


@pytest.mark.parametrize("V", [33, 64, 1024, 1025, 2047, 2048, 2049])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_short_rows(V, dtype):
    """NaN, infinities, masked and equal entries where a warp holds a row."""
    x = logits_of(12, V, V + 1, dtype=dtype)
    x[1, 3] = math.nan
    x[2, V - 1] = math.inf
    x[3] = -math.inf
    x[4, torch.randperm(V, generator=torch.Generator().manual_seed(V))[7:]] = -math.inf
    x[5, 0], x[5, 1:] = 1.0, torch.finfo(dtype).min
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7, 10:] = x[7, 0]
    x[8] = torch.arange(V) * -2.0 ** -7
    x[9] = -30.0
    x[9, V // 2] = 1.0
    x[10] = torch.finfo(dtype).max
    targets = torch.tensor([(i * 5) % V for i in range(10)] + [-1, V])
    for top in sorted({0, 1, 5, 20, 32, min(V, 33), min(V, 64)}):
        check(x[:, :V], targets.clamp(max=V - 1), top)
    assert mi.token_scores(x.to(DEV), targets.to(DEV), top=1).logprob[11].isnan()


def test_many_rows():
    x = logits_of(700, 1003, 3)
    check(x, torch.randint(0, 1003, (700,)), 20)


def test_masked_rows():
    x = logits_of(6, 32000, 5)
    allowed = torch.zeros_like(x, dtype=torch.bool)
    for i, k in enumerate([1, 3, 19, 20, 500]):  # fewer tokens than alternatives: masked ones fill the list, lowest index first
        allowed[i, torch.randperm(32000, generator=torch.Generator().manual_seed(i))[:k]] = True
    x = x.masked_fill(~allowed, -math.inf)       # the last row: nothing is allowed
    s = check(x, torch.tensor([0, 1, 2, 3, 4, 5]), 20)
    assert s.entropy[0] == 0.0 and s.top_logprobs[0, 0] == 0.0 and s.entropy[5].isnan()


def test_infinities_and_numbers_that_are_none():
    x = logits_of(5, 9000, 6)
    x[0, 8500] = math.nan
    x[1, 17] = math.inf
    x[2, 8999] = -math.nan
    x[3] = -math.inf
    check(x, torch.tensor([3, 17, 4, 5, 6]), 4)


def test_equal_values():
    x = torch.zeros(3, 20000)
    x[0, ::2] = -0.0  # equal to 0
    x[1, 15000:15010] = 1.0
    x[2] = torch.arange(20000).float() * -1e-3  # sorted: all of the best in one place
    check(x, torch.tensor([1, 15003, 19999]), 64)


def test_lowest_values_of_the_type():
    x = torch.full((2, 5000), torch.finfo(torch.float32).min)
    x[0, 77] = 0.0
    x[1, 4000:] = torch.finfo(torch.float32).max
    check(x, torch.tensor([77, 4001]), 5)


def test_peaked_rows_keep_their_digits():
    """A token with almost all the probability: 1 - p, not p, sets the entropy and its own log-probability."""
    x = torch.full((3, 40000), -30.0)
    x[0, 5], x[1, 39999], x[2, 20000] = 0.0, 2.0, -11.0
    targets = torch.tensor([5, 39999, 20000])
    s = check(x, targets, 2)
    lp, ent, _, _ = U.scores_ref(x, targets, 2)
    # relative to themselves: exponents are exact to 2^-24 * 2^5, the exponential to 2^-22, sums to 2^-17
    for got, want in ((s.logprob, lp), (s.entropy, ent)):
        assert ((got.cpu().double() - want).abs() <= 2.0 ** -16 * want.abs()).all()


def test_rows_of_wider_ones_and_targets_past_the_vocabulary():
    wide = logits_of(4, 1100, 8)
    x = wide.to(DEV)[:, 50:1050]
    s = mi.token_scores(x, torch.tensor([0, 999, 1000, -5], device=DEV), top=3)
    want = mi.token_scores(x.contiguous(), torch.tensor([0, 999, -1, -1], device=DEV), top=3)
    assert torch.equal(s.top_ids, want.top_ids) and torch.equal(s.entropy, want.entropy)
    assert torch.equal(s.logprob[:2], want.logprob[:2]) and s.logprob[2].isnan() and s.logprob[3] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first,pitch", [(0, 40008), (4, 40004), (1, 40008), (0, 40001), (2, 40002)])
def test_rows_that_begin_anywhere(dtype, first, pitch):
    """The same bits wherever a row lies: 16-byte copies, 4-byte copies, single entries."""
    wide = logits_of(3, pitch, 8, dtype=dtype).to(DEV)
    x = wide[:, first: first + 40000]
    t = torch.tensor([5, 39999, 77], device=DEV)
    s, want = mi.token_scores(x, t, top=20), mi.token_scores(x.contiguous(), t, top=20)
    check(x.cpu(), t.cpu(), 20)
    for a, b in zip((s.logprob, s.entropy, s.top_ids, s.top_logprobs), (want.logprob, want.entropy, want.top_ids, want.top_logprobs)):
        assert torch.equal(a, b)


def test_more_rows_than_a_call_takes():
    x = logits_of(3, 40, 4).repeat(22000, 1)
    check(x, torch.arange(66000) % 40, 2)


def test_no_rows():
    s = mi.token_scores(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.long, device=DEV), top=3)
    assert s.logprob.shape == (0,) and s.top_ids.shape == (0, 3)


def test_the_same_bits_alone_captured_and_on_another_stream():
    x = logits_of(9, 50257, 9).to(DEV)
    t = torch.arange(9, device=DEV)
    a = mi.token_scores(x, t, top=7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = mi.token_scores(x, t, top=7)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = mi.token_scores(x, t, top=7)
    g.replay()
    one = mi.token_scores(x[4:5], t[4:5], top=7)
    torch.cuda.synchronize()
    for y in (b, c):
        assert torch.equal(a.logprob, y.logprob) and torch.equal(a.entropy, y.entropy) and torch.equal(a.top_ids, y.top_ids) and torch.equal(a.top_logprobs, y.top_logprobs)
    assert torch.equal(a.logprob[4:5], one.logprob) and torch.equal(a.top_ids[4:5], one.top_ids)


def check_large(x, targets, top):
    """As check(), for log-probabilities of any size: a difference of two numbers and of that and the logarithm, 2^-24 of itself each."""
    s = mi.token_scores(x.to(DEV), targets.to(DEV), top=top)
    lp, ent, ids, lps = U.scores_ref(x, targets, top)
    assert s.top_ids.cpu().tolist() == ids.tolist()
    for got, want in ((s.logprob, lp), (s.entropy, ent), (s.top_logprobs, lps)):
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        tol = 2.0 ** -17 + 2.0 ** -15 * want.abs().clamp(max=16) + 2.0 ** -23 * want.abs()
        fin = want.isfinite()
        assert ((got - want).abs() <= tol)[fin].all(), ((got - want).abs() / tol)[fin].max()


FILLS = [-(2.0 ** 24), -1e8, -1e9, -(2.0 ** 30), -1.5e9, -1e10] + [-(10.0 ** e) for e in range(11, 31)] + [-3e38]


@pytest.mark.parametrize("T,V", [(3, 5000), (160, 5000), (3, 40000), (160, 40000)])  # one segment or several, joined by a cluster or by a second launch
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [0, 20])
def test_masks_of_any_finite_number(T, V, dtype, top):
    """A grammar that leaves tokens in one place only: the other segments of a row hold nothing but the mask's number."""
    few = logits_of(len(FILLS), 100, 13, dtype=dtype)
    rows = []
    for i, fill in enumerate(FILLS):
        row = torch.full((V,), fill).to(dtype)
        at = (0, V - 100, V // 2)[i % 3]
        row[at: at + 100] = few[i]
        rows.append((row, at + 7))
    for i, m in enumerate((1e10, -1e10, 3e9, 1e12)):  # rows whose own numbers are that large, a few steps of the type apart
        row = torch.full((V,), -3e38 if i % 2 else 0.9 * m - abs(m)).to(dtype)
        row[5: V: 977] = torch.tensor(m).to(dtype)
        row[11: V: 1999] = (torch.tensor(m) - abs(m) * torch.finfo(dtype).eps).to(dtype)
        rows.append((row, 5))
    rows.append((torch.full((V,), -1e11).to(dtype), 3))  # nothing but the mask
    n = len(rows)
    for first in range(0, n, T):  # T rows a call; of many, a few different ones and the first over and over
        take = [rows[i] for i in range(first, min(n, first + T))] + [rows[0]] * max(0, first + T - n)
        check_large(torch.stack([r for r, _ in take]), torch.tensor([t for _, t in take]), top)
