"""Pages of 8-bit keys and values on the GPU, operator by operator against plain 64-bit restatements (paged_util)."""
import math
import random

import pytest
import torch

import mistral_inference_b200 as mi
from mistral_inference_b200 import _abi_paged
from mistral_inference_b200.paged import check_status, empty_pool

from . import paged_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def assert_same_state(t: mi.PageTables, h: U.HostTables):
    assert t.table.tolist() == h.table and t.lens.tolist() == h.lens and t.free.tolist() == h.free and t.n_free.item() == h.n_free


# ---------------------------------------------------------------------------------------------------------------- plans
@pytest.mark.parametrize("adds", [[1], [0], [64], [63, 65, 1, 0, 128], [0, 0, 7, 0], [1] * 300, [1000, 3, 0, 700], [64] * 20, [5000, 1, 2500]])
@pytest.mark.parametrize("past", [0, 1, 63, 64, 100])
def test_extend_and_truncate(adds, past):
    B = len(adds)
    width = U.cdiv(past + max(adds) + 70, 64)
    n = sum(U.cdiv(past + a + 70, 64) for a in adds)
    t, h = mi.PageTables.empty(B, width, n, DEV), U.HostTables(B, width, n)
    for step in ([past] * B, adds, [1] * B):
        plan = t.extend(ints(step), sum(step)).check()
        positions, slots, q_start, seqpos = h.extend(step)
        assert plan.positions.tolist() == positions and plan.slots.tolist() == slots and plan.q_start.tolist() == q_start and plan.seqpos.tolist() == seqpos
        assert_same_state(t, h)
    check_status(t.truncate(ints([past] * B)))  # what the two steps took goes back ...
    h.truncate([past] * B)
    assert_same_state(t, h)
    t.extend(ints(adds), sum(adds)).check()     # ... and is found again
    h.extend(adds)
    assert_same_state(t, h)


def test_rows_in_any_order_and_requests_that_end():
    rnd = random.Random(3)
    R, width, n = 40, 12, 300
    t, h = mi.PageTables.empty(R, width, n, DEV), U.HostTables(R, width, n)
    for _ in range(30):
        rows = rnd.sample(range(R), rnd.randint(1, R))
        if rnd.random() < 0.4:
            keep = [rnd.choice([0, h.lens[r], rnd.randint(0, h.lens[r])]) for r in rows]
            check_status(t.truncate(ints(keep), ints(rows)))
            h.truncate(keep, rows)
        else:
            add = [min(rnd.choice([0, 1, rnd.randint(0, 130)]), width * 64 - h.lens[r]) for r in rows]
            room = sum(add) + rnd.choice([0, 0, 9])
            if sum(U.cdiv(h.lens[r] + a, 64) - U.cdiv(h.lens[r], 64) for r, a in zip(rows, add)) > h.n_free:
                continue
            plan = t.extend(ints(add), room, ints(rows)).check()
            positions, slots, q_start, seqpos = h.extend(add, rows)
            pad = room - sum(add)
            assert plan.positions.tolist() == positions + [0] * pad and plan.slots.tolist() == slots + [-1] * pad
            assert plan.q_start.tolist() == q_start and plan.seqpos.tolist() == seqpos
        assert_same_state(t, h)


def test_steps_that_cannot_be_done_change_nothing():
    t, h = mi.PageTables.empty(3, 4, 6, DEV), U.HostTables(3, 4, 6)
    t.extend(ints([100, 64, 1]), 165).check()
    h.extend([100, 64, 1])
    for add, room, rows, why in [([1, 1, 1], 3, [0, 1, 0], "twice"), ([1, 1, 1], 3, [0, 1, 3], "row"), ([1, 1, 1], 3, [-1, 1, 2], "row"), ([1, -1, 1], 3, None, "length"),
                                 ([157, 1, 1], 200, None, "length"), ([2 ** 31 - 1, 1, 1], 3, None, "length"), ([1, 1, 1], 2, None, "room"), ([100, 65, 64], 300, None, "free")]:
        plan = t.extend(ints(add), room, None if rows is None else ints(rows))
        with pytest.raises(_abi_paged.Mb200Error, match=why):
            plan.check()
        assert plan.q_start.tolist() == [0] * 4 and plan.slots.tolist() == [-1] * room
        assert_same_state(t, h)
    for keep, rows, why in [([101, 0, 0], None, "length"), ([-1, 0, 0], None, "length"), ([0, 0], [1, 1], "twice"), ([0], [7], "row")]:
        with pytest.raises(_abi_paged.Mb200Error, match=why):
            check_status(t.truncate(ints(keep), None if rows is None else ints(rows)))
        assert_same_state(t, h)


def test_a_row_named_twice_among_many_tokens():
    """Every CTA of the call finds it, and the next call starts afresh."""
    t, h = mi.PageTables.empty(40, 200, 8000, DEV), U.HostTables(40, 200, 8000)
    rows = [(7 * i) % 40 for i in range(40)]
    for i in range(10):
        twice = list(rows)
        twice[39] = rows[i]
        plan = t.extend(ints([1000] * 40), 40000, ints(twice))
        with pytest.raises(_abi_paged.Mb200Error, match="twice"):
            plan.check()
        assert plan.q_start.tolist() == [0] * 41 and (plan.slots == -1).all()
        assert_same_state(t, h)
        plan = t.extend(ints([900] * 40), 40000, ints(rows)).check()
        _, slots, _, _ = h.extend([900] * 40, rows)
        assert plan.slots.tolist() == slots + [-1] * 4000
        assert_same_state(t, h)


def test_tables_refuse_what_they_cannot_take():
    t = mi.PageTables.empty(2, 4, 8, DEV)
    with pytest.raises(AssertionError):
        t.extend(ints([1, 1, 1]), 3)  # more requests than rows
    with pytest.raises(AssertionError):
        t.extend(torch.ones(2, device=DEV), 2)
    with pytest.raises(AssertionError):
        t.extend(torch.ones(2, dtype=torch.int32), 2)
    with pytest.raises(AssertionError):
        t.extend(ints([1, 7, 1, 7])[::2], 2)
    with pytest.raises(AssertionError):
        t.truncate(ints([1, 1]), rows=ints([1]))
    with pytest.raises(_abi_paged.Mb200Error, match="requests"):
        big = mi.PageTables.empty(_abi_paged.MAX_REQUESTS + 1, 1, 8, DEV)
        big.extend(torch.zeros(_abi_paged.MAX_REQUESTS + 1, dtype=torch.int32, device=DEV), 0)


def test_many_requests_at_once():
    B = _abi_paged.MAX_REQUESTS
    t, h = mi.PageTables.empty(B, 2, 2 * B, DEV), U.HostTables(B, 2, 2 * B)
    rnd = random.Random(1)
    for _ in range(2):
        add = [rnd.randint(0, 60) for _ in range(B)]
        plan = t.extend(ints(add), sum(add)).check()
        positions, slots, q_start, _ = h.extend(add)
        assert plan.positions.tolist() == positions and plan.slots.tolist() == slots and plan.q_start.tolist() == q_start
    assert_same_state(t, h)
    check_status(t.truncate(ints([0] * B)))
    h.truncate([0] * B)
    assert_same_state(t, h)


@pytest.mark.parametrize("R", [129, 4000, 131072])
def test_few_requests_of_states_with_many_rows(R):
    """One or two requests of a state of many rows, the last ones among them: what marks a row as named has a place for every row."""
    t, h = mi.PageTables.empty(R, 2, 64, DEV), U.HostTables(R, 2, 64)
    def same():  # rows as tensors: a state of 131072 rows is slow as lists
        assert torch.equal(t.table.cpu(), torch.tensor(h.table, dtype=torch.int32)) and t.lens.tolist() == h.lens and t.free.tolist() == h.free and t.n_free.item() == h.n_free
    for add, rows in [([70], [R - 1]), ([3, 65], [R // 2, 0]), ([1], [R - 1]), ([5, 0], [R - 2, R - 1]), ([64], [127])]:
        plan = t.extend(ints(add), sum(add), ints(rows)).check()
        positions, slots, q_start, seqpos = h.extend(add, rows)
        assert plan.positions.tolist() == positions and plan.slots.tolist() == slots and plan.q_start.tolist() == q_start and plan.seqpos.tolist() == seqpos
        same()
    for rows in ([R - 1, R - 1], [R, 0], [0, -1]):
        with pytest.raises(_abi_paged.Mb200Error, match="row"):
            t.extend(ints([1, 1]), 2, ints(rows)).check()
        with pytest.raises(_abi_paged.Mb200Error, match="row"):
            check_status(t.truncate(ints([0, 0]), ints(rows)))
    for keep, rows in [([0], [R - 1]), ([2, 0], [R // 2, R - 2]), ([0], [127])]:
        check_status(t.truncate(ints(keep), ints(rows)))
        h.truncate(keep, rows)
        same()


def test_a_cache_of_many_rows_admits_and_retires_single_requests():
    c = mi.PagedCache(1, 1000, 256, 1, 128, n_pages=40)
    for i in range(6):
        places = c.admit(1)
        c.get_input_metadata([0] * places[0] + [10 + 30 * i])[0].plan.check()
        c.update_seqlens([0] * places[0] + [10 + 30 * i])
    c.retire([2])
    c.retire([0, 4])
    c.admit(2)
    c.get_input_metadata([1, 0, 1, 64, 0])[0].plan.check()
    c.update_seqlens([1, 0, 1, 64, 0])
    lens = c.tables.lens.tolist()
    assert [lens[r] for r in c.rows] == c.ledger.lens == [41, 100, 131, 64, 0] and sum(lens) == sum(c.ledger.lens)
    assert int(c.tables.n_free) == c.ledger.free_pages


# ---------------------------------------------------------------------------------------------------------------- writes
def numbers(*shape, seed, spread=4, dtype=torch.bfloat16):
    """Normal numbers of magnitudes that differ by token and head."""
    g = torch.Generator().manual_seed(seed)
    size = torch.exp2(torch.randint(-spread, spread + 1, (*shape[:-1], 1), generator=g).float())
    return (torch.randn(*shape, generator=g) * size).to(dtype)


class Pool:
    """A layer's pool on the GPU beside its 64-bit restatement."""

    def __init__(self, n_pages, KV):
        self.kv, self.scale = empty_pool(n_pages, KV, DEV)
        self.kv.view(torch.uint8).fill_(0x7F)  # NaN where nobody has written
        self.scale.fill_(2.0 ** 20)
        self.ref_kv, self.ref_scale = self.kv.cpu().double(), self.scale.cpu().double()

    def write(self, k, v, plan, slots):
        mi.write_pages(self.kv, self.scale, k, v, plan)
        U.write_ref(self.ref_kv, self.ref_scale, k.cpu(), v.cpu(), slots)

    def assert_same(self):
        assert torch.equal(self.scale.cpu().double(), self.ref_scale)
        got = self.kv.cpu().double()
        assert torch.equal(got.isnan(), self.ref_kv.isnan()) and torch.equal(got.nan_to_num(0.0), self.ref_kv.nan_to_num(0.0))


@pytest.mark.parametrize("KV", [1, 2, 8])
@pytest.mark.parametrize("steps", [[[1], [1], [1]], [[64], [1]], [[63, 1], [1, 0], [3, 70]], [[200, 3, 64, 0, 130], [1, 1, 1, 1, 1], [0, 200, 0, 5, 63]]])
def test_write(KV, steps):
    B = len(steps[0])
    total = [sum(s[b] for s in steps) for b in range(B)]
    n = sum(U.cdiv(x, 64) for x in total) + 2
    t, h, pool = mi.PageTables.empty(B, U.cdiv(max(total), 64), n, DEV), U.HostTables(B, U.cdiv(max(total), 64), n), Pool(n, KV)
    for i, step in enumerate(steps):
        plan = t.extend(ints(step), sum(step)).check()
        _, slots, _, _ = h.extend(step)
        k, v = numbers(sum(step), KV, 128, seed=i).to(DEV), numbers(sum(step), KV, 128, seed=50 + i).to(DEV)
        pool.write(k, v, plan, slots)
        pool.assert_same()
        mi.write_pages(pool.kv, pool.scale, k, v, plan)  # the same step again
        pool.assert_same()


def test_write_of_a_portion_among_single_tokens():
    """Few tokens a request on average, so a warp writes a page, whose rows it takes in turns; the earlier tokens' codes move to grown scales on the way."""
    B, KV = 40, 3
    t, h, pool = mi.PageTables.empty(B, 6, 3 * B, DEV), U.HostTables(B, 6, 3 * B), Pool(3 * B, KV)
    for i, step in enumerate([[1] * 20 + [37] + [1] * 19, [i % 3 for i in range(39)] + [200], [63] + [0] * 18 + [17, 130] + [1] * 19]):
        plan = t.extend(ints(step), sum(step)).check()
        _, slots, _, _ = h.extend(step)
        pool.write(numbers(sum(step), KV, 128, seed=i, spread=4 + 4 * i).to(DEV), numbers(sum(step), KV, 128, seed=50 + i, spread=4 + 4 * i).to(DEV), plan, slots)
        pool.assert_same()


def test_write_of_growing_shrinking_and_strange_numbers():
    t, h, pool = mi.PageTables.empty(1, 2, 3, DEV), U.HostTables(1, 2, 3), Pool(3, 2)
    values = [0.0, 1e-30, 1.0, 448.0, 450.0, 3e38, 0.0, -3.3e38, float("inf"), float("nan"), -float("inf"), 2.0, 2.0 ** -126, 2.0 ** -133]
    for i, x in enumerate(values):
        plan = t.extend(ints([1]), 1).check()
        _, slots, _, _ = h.extend([1])
        k = numbers(1, 2, 128, seed=i, spread=0).clamp(-1, 1)
        k[0, 0, 5] = x
        k[0, 1] = x
        pool.write(k.to(DEV), torch.flip(k, (1,)).contiguous().to(DEV), plan, slots)
        pool.assert_same()


def test_write_takes_rows_of_wider_matrices_and_leaves_empty_places_out():
    KV, T = 4, 70
    t, h, pool = mi.PageTables.empty(2, 2, 4, DEV), U.HostTables(2, 2, 4), Pool(4, KV)
    plan = t.extend(ints([60, 5]), T).check()  # five places stay empty
    _, slots, _, _ = h.extend([60, 5])
    qkv = numbers(T, 24 * 128, seed=4).to(DEV)
    k, v = qkv[:, 16 * 128: 20 * 128], qkv[:, 20 * 128:]
    mi.write_pages(pool.kv, pool.scale, k, v, plan)
    U.write_ref(pool.ref_kv, pool.ref_scale, k.cpu()[:65].reshape(65, KV, 128), v.cpu()[:65].reshape(65, KV, 128), slots)
    pool.assert_same()


def test_stacks_that_are_none():
    """A count of free pages that the stack cannot have is refused; an id that no pool has becomes no slot, and not another page's."""
    for n_free in (9, 2 ** 31 - 1, -1, -2 ** 31):
        t = mi.PageTables(torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ints([0, 0]), ints(list(range(8))), ints([n_free]))
        with pytest.raises(_abi_paged.Mb200Error, match="free"):
            t.extend(ints([70, 1]), 71).check()
        t.table[0, :2], t.lens[0] = ints([6, 7]), 100
        with pytest.raises(_abi_paged.Mb200Error, match="free"):
            check_status(t.truncate(ints([0, 0])))
        assert t.lens.tolist() == [100, 0] and t.free.tolist() == list(range(8)) and t.n_free.item() == n_free
    for page in (2 ** 25, 2 ** 25 + 1, 2 ** 31 - 1, -1):
        t = mi.PageTables(torch.full((1, 4), -1, dtype=torch.int32, device=DEV), ints([0]), ints([page, 3]), ints([2]))
        plan = t.extend(ints([70]), 70).check()
        assert plan.slots.tolist() == list(range(192, 256)) + [-1] * 6 and t.table.tolist() == [[3, page, -1, -1]]
        pool, k = Pool(4, 1), numbers(70, 1, 128, seed=1)
        pool.write(k.to(DEV), k.to(DEV), plan, plan.slots.tolist())
        pool.assert_same()
        out = mi.attend_pages(k.to(DEV), pool.kv, pool.scale, plan)
        assert out[:64].isfinite().all() and out[64:].isnan().all()


# ---------------------------------------------------------------------------------------------------------------- attention
def filled(KV, past, new, seed, extra_rows=0, kv_std=1.0):
    """(tables' plan of `new` tokens behind `past`, pool) with pages in a random order and random codes everywhere; what nobody has written is NaN."""
    rnd = random.Random(seed)
    B = len(past)
    total = [p + n for p, n in zip(past, new)]
    width = U.cdiv(max(total), 64) + 1
    n = sum(U.cdiv(x, 64) for x in total) + 3
    order = list(range(n))
    rnd.shuffle(order)
    t = mi.PageTables(torch.full((B + extra_rows, width), -1, dtype=torch.int32, device=DEV), torch.zeros(B + extra_rows, dtype=torch.int32, device=DEV), ints(order), ints([n]))
    rows = rnd.sample(range(B + extra_rows), B)
    t.extend(ints(past), sum(past), ints(rows)).check()
    plan = t.extend(ints(new), sum(new), ints(rows), longest=max(new), most=max(total)).check()
    g = torch.Generator().manual_seed(seed)
    kv = (torch.randn(n, KV, 2, 64, 128, generator=g) * kv_std * 60).clamp(-448, 448).to(U.E4M3)
    scale = torch.exp2(torch.randint(-8, -4, (n, KV, 2), generator=g).float())
    table = t.table.cpu().tolist()
    held = torch.zeros(n, 64, dtype=torch.bool)
    for r, x in zip(rows, total):
        for pos in range(x):
            held[table[r][pos // 64], pos % 64] = True
    raw = kv.view(torch.uint8)
    raw[(~held)[:, None, None].expand(-1, KV, 2, -1)] = 0x7F
    return plan, kv.to(DEV), scale.to(DEV), kv, scale, table, rows


def check_attention(H, KV, past, new, window=0, seed=0, q_scale=1.0, softmax_scale=None, kv_std=1.0, **kw):
    plan, kv, scale, kv_h, scale_h, table, rows = filled(KV, past, new, seed, kv_std=kv_std)
    T = sum(new)
    q = (torch.randn(T, H, 128, generator=torch.Generator().manual_seed(seed + 1)) * q_scale).to(torch.bfloat16)
    got = mi.attend_pages(q.to(DEV), kv, scale, plan, window=window, softmax_scale=softmax_scale, **kw)
    plan.check()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    want, mag = U.attend_ref(q, kv_h.double(), scale_h, table, rows, starts, past, window, softmax_scale)
    got = got.cpu().double().view(T, H, 128)
    tol = U.attend_tolerance(want, mag, max(p + n for p, n in zip(past, new)), float(448 * scale_h.max()))
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1, f"{worst:.2f} times the tolerance"
    return got


@pytest.mark.parametrize("H,KV", [(4, 4), (4, 2), (8, 2), (12, 2), (8, 1), (16, 1), (32, 1), (9, 3), (32, 8)])
@pytest.mark.parametrize("past", [[0], [1, 63, 64], [127, 128, 129, 500]])
def test_attention_of_single_tokens(H, KV, past):
    check_attention(H, KV, past, [1] * len(past), seed=len(past))


@pytest.mark.parametrize("past", [[1000], [2047, 5], [4100, 1, 0, 300]])
@pytest.mark.parametrize("window", [0, 1, 64, 65, 1000])
def test_attention_of_single_tokens_in_windows(past, window):
    check_attention(8, 2, past, [1] * len(past), window=window, seed=window)


@pytest.mark.parametrize("new", [[2], [5, 1, 3], [0, 4, 0], [17], [33, 2], [64, 70], [130, 1, 0, 7]])
@pytest.mark.parametrize("H,KV,window", [(8, 2, 0), (12, 2, 0), (4, 4, 50), (16, 1, 100)])
def test_attention_of_several_tokens(new, H, KV, window):
    check_attention(H, KV, [0, 100, 63, 200][: len(new)], new, window=window, seed=len(new))


def by_rings(H, KV, past, new, window=0):
    """Whether such a call's pages go through 16-bit rings."""
    total = [p + n for p, n in zip(past, new)]
    return _abi_paged.lib().mbp_attn_pages_scratch(len(past), sum(new), max(new), max(total), U.cdiv(max(total), 64) + 1, H, KV, window) > 0


@pytest.mark.parametrize("H,KV,past,new,window", [(32, 8, [0, 300], [300, 129], 0), (16, 16, [100, 0, 63], [500, 300, 0], 0), (24, 8, [700, 64], [200, 333], 150), (8, 1, [1000, 0, 5, 64], [400, 1, 130, 77], 65),
                                                  (15, 5, [200, 100], [550, 460], 0), (32, 8, [1500, 3], [190, 333], 1000)])
def test_attention_of_portions(H, KV, past, new, window):
    assert by_rings(H, KV, past, new, window)
    check_attention(H, KV, past, new, window=window, seed=len(new))


def test_portions_of_one_request_at_a_time():
    """Rings of a gigabyte at most: requests take turns, and a `most` of 0 stands for the whole row of the block table."""
    plan, kv, scale, *_ = filled(8, [100, 30, 7], [250, 300, 200], 4)
    q = numbers(750, 32, 128, seed=1, spread=0).to(DEV)
    want = mi.attend_pages(q, kv, scale, plan)
    wide = torch.full((plan.table.shape[0], 4200), -1, dtype=torch.int32, device=DEV)
    wide[:, : plan.table.shape[1]] = plan.table
    loose = mi.PagePlan(wide, plan.rows, plan.q_start, plan.seqpos, plan.positions, plan.slots, plan.longest)
    assert _abi_paged.lib().mbp_attn_pages_scratch(3, 900, 300, 0, 4200, 32, 8, 0) == 4200 * 64 * 8 * 128 * 4 > 1 << 30
    assert torch.equal(mi.attend_pages(q, kv, scale, loose), want)


def test_portions_longer_than_the_plan_says_are_no_numbers():
    plan, kv, scale, *_ = filled(8, [900, 30], [250, 300], 4)
    q = numbers(550, 32, 128, seed=1, spread=0).to(DEV)
    want = mi.attend_pages(q, kv, scale, plan)
    plan.check()
    plan.most = 400
    got = mi.attend_pages(q, kv, scale, plan)
    assert got[:250].isnan().all() and torch.equal(got[250:], want[250:])
    with pytest.raises(_abi_paged.Mb200Error, match="most"):
        plan.check()


@pytest.mark.parametrize("KV,past,new,longest", [(8, [900, 30], [250, 300], 260), (8, [900, 30], [250, 300], 200), (2, [900, 30], [250, 300], 260), (2, [70, 30, 5], [1, 3, 2], 1),
                                                 (2, [70, 30], [40, 12], 12)])
def test_requests_that_bring_more_than_the_plan_says(KV, past, new, longest):
    """Both ways of attending: what there is no room for is no number, the other requests are right."""
    plan, kv, scale, kv_h, scale_h, table, rows = filled(KV, past, new, 4)
    T, H = sum(new), 4 * KV
    q = numbers(T, H, 128, seed=1, spread=0)
    plan.longest = longest
    got = mi.attend_pages(q.to(DEV), kv, scale, plan, out=torch.full((T, H * 128), 9.0, dtype=torch.bfloat16, device=DEV)).cpu().double().view(T, H, 128)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    want, mag = U.attend_ref(q, kv_h.double(), scale_h, table, rows, starts, past)
    tol = U.attend_tolerance(want, mag, max(p + n for p, n in zip(past, new)), float(448 * scale_h.max()))
    gone = got.isnan().all(2).all(1)
    assert torch.equal(gone, got.isnan().any(2).any(1)) and ((got - want).abs() <= tol)[~gone].all()
    for b, n in enumerate(new):
        assert not gone[starts[b]: starts[b] + n].any() if n <= longest else gone[starts[b] + n - 1]
    with pytest.raises(_abi_paged.Mb200Error, match="longest"):
        plan.check()


def test_portions_of_pages_that_are_none_and_of_refused_plans():
    plan, kv, scale, *_ = filled(8, [200, 30], [250, 300], 4)
    q = numbers(550, 32, 128, seed=1, spread=0).to(DEV)
    want = mi.attend_pages(q, kv, scale, plan)
    for page in (-1, kv.shape[0], 2 ** 30):
        table = plan.table.clone()
        table[int(plan.rows[0]), 0] = page
        got = mi.attend_pages(q, kv, scale, mi.PagePlan(table, plan.rows, plan.q_start, plan.seqpos, plan.positions, plan.slots, plan.longest, plan.most))
        assert got[:250].isnan().all() and torch.equal(got[250:], want[250:])
    t = mi.PageTables.empty(2, 8, 3, DEV)
    refused = t.extend(ints([250, 300]), 550, longest=300, most=300)
    out = torch.full((550, 32 * 128), 3.0, dtype=torch.bfloat16, device=DEV)
    mi.attend_pages(q, kv, scale, refused, out=out)
    mi.write_pages(kv.clone(), scale.clone(), q[:, :8].contiguous(), q[:, :8].contiguous(), refused)
    assert (out == 3.0).all()


@pytest.mark.parametrize("H,KV,rings", [(32, 8, True), (8, 2, False)])
def test_plans_that_name_rows_that_are_not_there(H, KV, rings):
    """Both ways of attending: a request whose tokens reach behind the queries, or that begins before position 0, is left out; nothing is written elsewhere."""
    plan, kv, scale, *_ = filled(KV, [200, 30], [250, 300], 4)
    assert by_rings(H, KV, [200, 30], [250, 300]) == rings
    q = numbers(550, H, 128, seed=1, spread=0).to(DEV)
    want = mi.attend_pages(q, kv, scale, plan)
    for q_start, seqpos in (([0, 250, 551], [200, 30]), ([0, 250, 900], [200, 30]), ([0, 250, 550], [200, -1]), ([0, 250, 550], [200, -2 ** 31]), ([0, 250, 2 ** 31 - 1], [200, 30])):
        room = torch.full((1200, H * 128), 3.0, dtype=torch.bfloat16, device=DEV)
        odd = mi.PagePlan(plan.table, plan.rows, ints(q_start), ints(seqpos), plan.positions, plan.slots, plan.longest, plan.most)
        mi.attend_pages(q, kv, scale, odd, out=room[:550])
        assert torch.equal(room[:250], want[:250]) and (room[250:] == 3.0).all()


def test_portions_out_of_a_wider_matrix():
    plan, kv, scale, kv_h, scale_h, table, rows = filled(8, [200, 30], [250, 300], 4)
    wide = numbers(550, 48 * 128, seed=1, spread=0).to(DEV)
    for first in (0, 8, 1024):
        x = wide[:, first: first + 32 * 128]
        assert torch.equal(mi.attend_pages(x, kv, scale, plan), mi.attend_pages(x.contiguous(), kv, scale, plan))
    x = numbers(550, 33 * 128 + 4, seed=1, spread=0).to(DEV)[:, 4: 4 + 32 * 128]  # rows that the copy engine cannot take
    got = mi.attend_pages(x, kv, scale, plan).cpu().double().view(550, 32, 128)
    want, mag = U.attend_ref(x.cpu().reshape(550, 32, 128), kv_h.double(), scale_h, table, rows, [0, 250, 550], [200, 30])
    assert ((got - want).abs() <= U.attend_tolerance(want, mag, 450, float(448 * scale_h.max()))).all()


@pytest.mark.parametrize("q_scale", [1e-3, 30.0])
def test_attention_of_small_and_large_queries(q_scale):
    """Nearly even weights, and weights that one key has almost alone."""
    check_attention(8, 2, [300, 64], [1, 3], seed=5, q_scale=q_scale, kv_std=0.3)


def test_attention_with_a_scale_of_its_own_and_into_rows_of_the_caller():
    out = torch.full((4, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    got = check_attention(8, 2, [90, 10], [3, 1], seed=6, softmax_scale=0.03, out=out)
    assert torch.equal(out.cpu().double().view(4, 8, 128), got)


def test_attention_leaves_rows_behind_the_last_token():
    plan, kv, scale, *_ = filled(2, [70, 3], [1, 1], 3)
    padded = mi.PagePlan(plan.table, plan.rows, plan.q_start, plan.seqpos, torch.cat([plan.positions, ints([0, 0])]), torch.cat([plan.slots, ints([-1, -1])]), 1, plan.most)
    q = numbers(4, 8, 128, seed=1, spread=0).to(DEV)
    out = torch.full((4, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    mi.attend_pages(q, kv, scale, padded, out=out)
    assert (out[2:] == 7.0).all() and torch.equal(out[:2], mi.attend_pages(q[:2], kv, scale, plan))


def test_attention_takes_queries_out_of_a_wider_matrix():
    plan, kv, scale, *_ = filled(2, [70, 3], [2, 1], 3)
    qkv = numbers(3, 12 * 128, seed=1, spread=0).to(DEV)
    assert torch.equal(mi.attend_pages(qkv[:, :1024], kv, scale, plan), mi.attend_pages(qkv[:, :1024].contiguous().view(3, 8, 128), kv, scale, plan))


def test_numbers_that_are_none_stay_with_the_queries_that_see_them():
    """NaN in keys or values: queries that see it are NaN, in every column of values or in that one; others are what they were."""
    plan, kv, scale, *_ = filled(2, [300, 200], [1, 1], 9)
    q = numbers(2, 8, 128, seed=2, spread=0).to(DEV)
    clean = mi.attend_pages(q, kv, scale, plan)
    page = int(plan.table[int(plan.rows[0]), 1])
    bad = kv.view(torch.uint8).clone()
    bad[page, 1, 1, 7, 33] = 0x7F  # a value of the first request's second key/value head
    got = mi.attend_pages(q, bad.view(U.E4M3), scale, plan).view(2, 8, 128)
    hit = got.isnan()
    assert hit[0, 4:, 33].all() and hit.sum() == 4
    assert torch.equal(got[~hit], clean.view(2, 8, 128)[~hit])
    got = mi.attend_pages(q, bad.view(U.E4M3), scale, plan, window=301 - 72)  # positions from 72 on: not the one at 71
    assert not got.isnan().any()
    bad = kv.view(torch.uint8).clone()
    bad[page, 1, 0, 7, 33] = 0x7F  # a key
    got = mi.attend_pages(q, bad.view(U.E4M3), scale, plan).view(2, 8, 128)
    assert got[0, 4:].isnan().all() and got.isnan().sum() == 4 * 128


@pytest.mark.parametrize("past,new,window", [(300, 5, 0), (60, 8, 0), (125, 8, 0), (300, 6, 40), (61, 7, 3), (2, 8, 20), (130, 8, 8), (190, 2, 64)])
def test_values_that_are_none_stay_with_the_tokens_that_see_them(past, new, window):
    """Several tokens at once: those before a NaN, and those whose window has left it behind, do not notice."""
    plan, kv, scale, *_ = filled(2, [past, 40], [new, 1], 9)
    q = numbers(new + 1, 8, 128, seed=2, spread=0).to(DEV)
    clean = mi.attend_pages(q, kv, scale, plan, window=window).view(new + 1, 8, 128)
    for at in sorted({past - 1, past, past + 1, past + new // 2, past + new - 1, max(0, past - window + 1), max(0, past - window + new // 2 + 1)}):
        for code, dim in ((0x7F, 33), (0xFF, 126)):
            bad = kv.view(torch.uint8).clone()
            bad[int(plan.table[int(plan.rows[0]), at // 64]), 1, 1, at % 64, dim] = code
            got = mi.attend_pages(q, bad.view(U.E4M3), scale, plan, window=window).view(new + 1, 8, 128)
            want = torch.zeros_like(got, dtype=torch.bool)
            for i in range(new):
                want[i, 4:, dim] = at <= past + i and (window == 0 or at > past + i - window)
            assert torch.equal(got.isnan(), want), (at, code)
            assert torch.equal(got[~want], clean[~want])


def test_pages_that_are_none_make_no_numbers():
    plan, kv, scale, *_ = filled(2, [300, 200], [1, 1], 9)
    q = numbers(2, 8, 128, seed=2, spread=0).to(DEV)
    clean = mi.attend_pages(q, kv, scale, plan)
    for page in (-1, kv.shape[0], 2 ** 30):
        table = plan.table.clone()
        table[int(plan.rows[0]), 2] = page
        got = mi.attend_pages(q, kv, scale, mi.PagePlan(table, plan.rows, plan.q_start, plan.seqpos, plan.positions, plan.slots, 1, plan.most))
        assert got[0].isnan().all() and torch.equal(got[1], clean[1])
    rows = plan.rows.clone()
    rows[0] = 99
    got = mi.attend_pages(q, kv, scale, mi.PagePlan(plan.table, rows, plan.q_start, plan.seqpos, plan.positions, plan.slots, 1, plan.most))
    assert got[0].isnan().all() and torch.equal(got[1], clean[1])


def test_the_same_bits_every_time():
    plan, kv, scale, *_ = filled(2, [3000, 100], [1, 1], 11)
    q = numbers(2, 8, 128, seed=2, spread=0).to(DEV)
    a = mi.attend_pages(q, kv, scale, plan)
    for _ in range(5):
        assert torch.equal(a, mi.attend_pages(q, kv, scale, plan))


@pytest.mark.parametrize("gap", [10.0, 16.0, 20.0, 21.5, 22.06, 22.5, 24.0, 60.0])
@pytest.mark.parametrize("H,new,at", [(8, 1, 0), (8, 1, 20000), (32, 4, 100)])
def test_many_small_weights_beside_a_large_one(gap, H, new, at):
    """One key `gap` binary places above tens of thousands of equal ones whose values share a sign: each of those weighs next to nothing, all of them together do not.  Many requests, so that
    one CTA walks over all keys of a request (they are one request's pages, named by all).  Weights: 2^-8 of themselves, or 2^-22 of the weight that they are held against: the largest
    so far for a CTA's first 2048 keys (2^-11 of the values' largest in all), then one at most 2^8 above the largest of their tile, whose others here are as large: 2^-14 of themselves.
    Scores and the result's rounding as in attend_tolerance."""
    KV, keys = 2, 30000 + new
    n = U.cdiv(keys, 64)
    g = torch.Generator().manual_seed(3)
    kv = torch.zeros(n, KV, 2, 64, 128)
    kv[:, :, 1] = 1.0 + torch.randint(0, 8, (n, KV, 64, 128), generator=g) / 8  # values in [1, 2)
    kv[at // 64, :, 0, at % 64, 0] = 1.0                                        # the large key, whose values are 0
    kv[at // 64, :, 1, at % 64] = 0.0
    kv, scale = kv.to(U.E4M3), torch.ones(n, KV, 2)
    q = torch.zeros(new, H, 128)
    q[:, :, 0] = gap / (128 ** -0.5 * math.log2(math.e))
    q = q.to(torch.bfloat16)
    B = 80
    plan = mi.PagePlan(torch.arange(n, dtype=torch.int32, device=DEV)[None].contiguous(), ints([0] * B), ints([new * b for b in range(B + 1)]), ints([30000] * B), ints([0] * new * B), ints([0] * new * B),
                       new, keys)
    assert not by_rings(H, KV, [30000] * B, [new] * B)
    got = mi.attend_pages(q.repeat(B, 1, 1).to(DEV), kv.to(DEV), scale.to(DEV), plan).cpu().double().view(B, new, H, 128)
    want, mag = U.attend_ref(q, kv.double(), scale, [list(range(n))], [0], [0, new], [30000])
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9 + 2.0 ** -14) * mag + 2.0 ** -11 * 2.0
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1, f"{worst:.2f} times the tolerance"


# ---------------------------------------------------------------------------------------------------------------- together
def test_a_run_of_requests_together():
    """Prompts, decode steps, drafts taken back, a request that ends and another that takes its pages: attention over what was written, at each step against 64 bits."""
    KV, H, R, width, n = 2, 8, 4, 6, 14
    t, h, pool = mi.PageTables.empty(R, width, n, DEV), U.HostTables(R, width, n), Pool(n, KV)
    seed = 0
    for what, rows, count in [("new", [0, 1], [100, 63]), ("new", [2], [70]), ("new", [0, 1, 2], [1, 1, 1]), ("new", [0, 1, 2], [4, 4, 4]), ("keep", [0, 1, 2], [102, 65, 72]),
                              ("new", [0, 1, 2], [1, 1, 1]), ("keep", [1], [0]), ("new", [3], [130]), ("new", [0, 2, 3], [1, 1, 1]), ("keep", [0], [64]), ("new", [0, 3], [2, 60])]:
        if what == "keep":
            check_status(t.truncate(ints(count), ints(rows)))
            h.truncate(count, rows)
            continue
        plan = t.extend(ints(count), sum(count), ints(rows), longest=max(count)).check()
        _, slots, q_start, seqpos = h.extend(count, rows)
        seed += 1
        k, v = numbers(sum(count), KV, 128, seed=seed, spread=1).to(DEV), numbers(sum(count), KV, 128, seed=seed + 100, spread=1).to(DEV)
        q = numbers(sum(count), H, 128, seed=seed + 200, spread=0).to(DEV)
        pool.write(k, v, plan, slots)
        got = mi.attend_pages(q, pool.kv, pool.scale, plan, window=90).cpu().double().view(-1, H, 128)
        pool.assert_same()
        want, mag = U.attend_ref(q.cpu(), pool.ref_kv.nan_to_num(0.0), pool.ref_scale, h.table, rows, q_start, seqpos, 90)
        tol = U.attend_tolerance(want, mag, 90, float(448 * pool.ref_scale[pool.ref_scale < 2.0 ** 20].max()))
        assert ((got - want).abs() <= tol).all()
    assert_same_state(t, h)


def test_captured_steps():
    """A decode step (plan, write, attention) in a graph: replays go on where the last one ended, on another stream too."""
    KV, H, B = 2, 8, 3
    t, eager = mi.PageTables.empty(B, 4, 12, DEV), mi.PageTables.empty(B, 4, 12, DEV)
    pools = [empty_pool(12, KV, DEV) for _ in range(2)]
    one, k, v, q = ints([1] * B), *(numbers(B, h, 128, seed=h, spread=0).to(DEV) for h in (KV, KV, H))

    def step(tables, pool, k, v, q):
        plan = tables.extend(one, B, longest=1)
        mi.write_pages(*pool, k, v, plan)
        return plan, mi.attend_pages(q, *pool, plan)

    for tables, pool in ((t, pools[0]), (eager, pools[1])):
        tables.extend(ints([62, 5, 100]), 167).check()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        keep = t.lens.clone()
        step(t, pools[0], k, v, q)  # warm-up, taken back
        t.truncate(keep)
        pools[0][0].view(torch.uint8).zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step(t, pools[0], k, v, q)
    for i in range(5):
        new = [numbers(B, h, 128, seed=10 * i + h, spread=2).to(DEV) for h in (KV, KV, H)]
        for dst, src in zip((k, v, q), new):
            dst.copy_(src)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        plan.check()
        _, want = step(eager, pools[1], *new)
        assert torch.equal(out, want) and t.lens.tolist() == eager.lens.tolist() == [62 + i + 1, 5 + i + 1, 100 + i + 1]


def test_two_states_on_two_streams():
    KV, H = 2, 8
    sides = [torch.cuda.Stream() for _ in range(2)]
    made = [filled(KV, [2000, 77], [1, 1], seed=s) for s in range(2)]
    q = numbers(2, H, 128, seed=3, spread=0).to(DEV)
    want = [mi.attend_pages(q, m[1], m[2], m[0]) for m in made]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                got[i].append(mi.attend_pages(q, made[i][1], made[i][2], made[i][0]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_a_pool_past_32_bit_offsets():
    """Pages behind the first 4 GB of a pool."""
    n, KV = 40000, 8  # 40000 * 8 * 16 KB = 5.2 GB
    kv = torch.zeros(n, KV, 2, 64, 128, dtype=torch.uint8, device=DEV).view(U.E4M3)
    scale = torch.ones(n, KV, 2, device=DEV)
    t = mi.PageTables(torch.full((1, 4), -1, dtype=torch.int32, device=DEV), ints([0]), ints([5, 39999, 33000, 39000]), ints([4]))
    plan = t.extend(ints([200]), 200).check()
    k, v, q = (numbers(200, h, 128, seed=h, spread=1).to(DEV) for h in (KV, KV, 8))
    mi.write_pages(kv, scale, k, v, plan)
    got = mi.attend_pages(q, kv, scale, plan)
    small = [5, 39999, 33000, 39000]
    kv2, scale2 = kv.view(torch.uint8)[small].contiguous().view(U.E4M3), scale[small].contiguous()
    assert float(scale2.min()) < 1 and not torch.equal(kv2.view(torch.uint8)[0], kv2.view(torch.uint8)[1])
    t2 = mi.PageTables(torch.full((1, 4), -1, dtype=torch.int32, device=DEV), ints([0]), ints([0, 1, 2, 3]), ints([4]))
    plan2 = t2.extend(ints([200]), 200).check()
    assert torch.equal(got, mi.attend_pages(q, kv2, scale2, plan2))
    check = kv.view(torch.uint8)[plan2.slots.long()[:1] // 64]
    assert check is not None


def test_writes_past_32_bit_offsets():
    """The same tokens into pages behind the first 4 GB and into a small pool: the same codes and scales, and nothing in between."""
    n, KV, ids = 40000, 8, [5, 39999, 33000, 39000]
    kv = torch.zeros(n, KV, 2, 64, 128, dtype=torch.uint8, device=DEV)
    scale = torch.ones(n, KV, 2, device=DEV)
    t = mi.PageTables(torch.full((1, 4), -1, dtype=torch.int32, device=DEV), ints([0]), ints(ids), ints([4]))
    small = mi.PageTables(torch.full((1, 4), -1, dtype=torch.int32, device=DEV), ints([0]), ints([0, 1, 2, 3]), ints([4]))
    pool = Pool(4, KV)
    pool.kv.view(torch.uint8).zero_()
    pool.scale.fill_(1.0)
    pool.ref_kv.zero_()
    pool.ref_scale.fill_(1.0)
    for i, count in enumerate((150, 1, 90)):
        k, v = (numbers(count, KV, 128, seed=2 * i + j, spread=1 + i).to(DEV) for j in range(2))
        mi.write_pages(kv, scale, k, v, t.extend(ints([count]), count).check())
        plan = small.extend(ints([count]), count).check()
        pool.write(k, v, plan, plan.slots.tolist())
    pool.assert_same()
    assert torch.equal(kv[ids], pool.kv.view(torch.uint8)) and torch.equal(scale[ids], pool.scale)
    kv[ids], scale[ids] = 0, 1.0
    assert int(kv.view(torch.int64).count_nonzero()) == 0 and (scale == 1.0).all()
