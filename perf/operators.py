"""Operators of serving requests of different lengths from a pool of 8-bit pages, as cases that can be timed and checked:

  plan    block tables and slot maps built on the GPU from request lengths
  write   keys and values of new tokens into pages of e4m3 numbers, one scale (a power of two) for each page, head and kind
  attend  causal attention of new tokens over the pages: one token a sequence, drafts of a few, portions of prompts
  score   log-probabilities of given tokens with the entropy of their distribution and the most likely alternatives

A page holds 64 tokens.  Pools are [pages, kv heads, 2 (keys, values), 64, 128] of e4m3 numbers beside [pages, kv heads, 2] scales; row r of a block table names the
pages of request r in order, -1 behind them; the free pages are a stack.  Shapes are those of this repository's configurations and generic ones."""
import math
import types
import zlib

import torch

own = False

DEV = "cuda"
HD = 128
PAGE = 64
E4M3_MAX = 448.0
LOWEST_EXP = -100  # exponent of the scale of a page of zeros

# query heads, key/value heads, window (0: none), vocabulary
SHAPES = {"7b": (32, 8, 4096, 32000), "nemo": (32, 8, 0, 131072), "8x22b": (48, 8, 0, 32768), "mha": (16, 16, 0, 32768), "w2048": (16, 4, 0, 32768), "narrow": (8, 1, 0, 1003)}


def listed():
    return [
        # a server's decode step of eight requests: one token each, few of them cross into a new page (nothing but latency)
        {"name": "plan_step_b8", "kind": "plan", "batch": 8, "new": 1, "past": 1500},
        # 64 prompts of very different lengths taken in at once
        {"name": "plan_prompts_b64", "kind": "plan", "batch": 64, "new": 1000, "past": 0},
        # the keys and values of one decode step of 32 requests, pages begun and half full
        {"name": "write_step_b32", "kind": "write", "shape": "nemo", "batch": 32, "new": 1, "past": 1106},
        # portions of three prompts behind what they have in the cache already
        {"name": "write_prompts_b3", "kind": "write", "shape": "7b", "batch": 3, "new": 2777, "past": 777},
        # chat with one user: one token over a full 4096-token window
        {"name": "attend_7b_b1", "kind": "attend", "shape": "7b", "batch": 1, "new": 1, "past": 5000},
        # a server's decode step: 32 requests of about 1100 tokens
        {"name": "attend_nemo_b32", "kind": "attend", "shape": "nemo", "batch": 32, "new": 1, "past": 1106},
        # four long documents that are being asked about
        {"name": "attend_long_b4", "kind": "attend", "shape": "nemo", "batch": 4, "new": 1, "past": 32500},
        # drafted tokens of eight requests verified at once, six query heads to a key/value head
        {"name": "attend_drafts_b8", "kind": "attend", "shape": "8x22b", "batch": 8, "new": 5, "past": 2100},
        # the fourth portion of three prompts (generate's chunk_size)
        {"name": "attend_portion_b3", "kind": "attend", "shape": "7b", "batch": 3, "new": 777, "past": 2331},
        # the answer's next token for one user: its log-probability beside five alternatives
        {"name": "score_7b_t1", "kind": "score", "vocab": 32000, "tokens": 1, "top": 5, "dtype": "fp32", "masked": 0},
        # a decode step of 32 requests whose answers are held to a grammar: most tokens are masked
        {"name": "score_masked_b32", "kind": "score", "vocab": 131072, "tokens": 32, "top": 20, "dtype": "fp32", "masked": 1},
        # scoring given text: a block of rows of the Nemo shape's head
        {"name": "score_nemo_t1000", "kind": "score", "vocab": 131072, "tokens": 1000, "top": 8, "dtype": "fp32", "masked": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "write", "attend", "attend", "attend", "score", "score"])
    if kind == "plan":
        new = rng.choice([1, _log(rng, 2, 1000)])
        return {"kind": kind, "batch": _log(rng, 1, 64 if new > 64 else 300), "new": new, "past": rng.choice([0, _log(rng, 1, 4000)])}
    shape = rng.choice(sorted(SHAPES))
    if kind == "write":
        new = rng.choice([1, _log(rng, 2, 2777)])
        return {"kind": kind, "shape": shape, "batch": _log(rng, 1, 3 if new > 300 else 48), "new": new, "past": rng.choice([0, _log(rng, 1, 1500)])}
    if kind == "attend":
        new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 700)])
        past = _log(rng, 1, 30000 if new <= 16 else 2331)
        batch = _log(rng, 1, max(1, min(48, 120000 // past))) if new <= 16 else rng.randint(1, 3)
        return {"kind": kind, "shape": shape, "batch": batch, "new": new, "past": past}
    vocab = rng.choice([1003, 32000, 32768, 50257, 131072])
    return {"kind": kind, "vocab": vocab, "tokens": rng.choice([_log(rng, 1, 64), _log(rng, 1, 100000000 // vocab // 2)]) if vocab > 2000 else _log(rng, 1, 4000),
            "top": rng.choice([1, 5, 20, 32]), "dtype": rng.choice(["fp32", "fp32", "bf16"]), "masked": rng.choice([0, 0, 1])}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed, name):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003) ^ zlib.crc32(name.encode()))


def _normal(seed, name, shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=_generator(seed, name))


def _new(case):
    """Tokens that each request brings: one each, or ragged below case["new"], the last request with the fewest."""
    n, b = case["new"], case["batch"]
    return [max(1, n - (i * n) // (2 * b)) for i in range(b)]


def _past(case):
    """Tokens that each request has in its pages: the first exactly case["past"], the others up to a quarter fewer."""
    n, b = case["past"], case["batch"]
    return [n - (i * n) // (4 * b) for i in range(b)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(tokens):
    return -(-tokens // PAGE)


def prepare(case, seed):
    st = types.SimpleNamespace(case=case)
    if case["kind"] == "score":
        T, V = case["tokens"], case["vocab"]
        # the head's logits are numbers of 16 bits, whatever they are kept in: equal ones are common
        st.logits = _normal(seed, "logits", (T, V), 2.5).to(torch.float32 if case["dtype"] == "fp32" else torch.bfloat16)
        st.targets = torch.randint(0, V, (T,), device=DEV, generator=_generator(seed, "targets"))
        if case["masked"]:  # a grammar: one token in a hundred is allowed, the target and the first among them
            allowed = torch.empty((T, V), device=DEV).uniform_(0, 1, generator=_generator(seed, "allowed")) < 0.01
            allowed.scatter_(1, st.targets[:, None], True)
            allowed[:, 0] = True
            st.logits.masked_fill_(~allowed, -math.inf)
        if T > 2:
            st.targets[T // 2] = -1  # the last token of a text has none to be scored for
        return st
    new, past, B = _new(case), _past(case), case["batch"]
    width = _pages(max(p + n for p, n in zip(past, new))) + 1
    used = [_pages(p) for p in past]
    total = sum(_pages(p + n) for p, n in zip(past, new)) + 7
    order = torch.randperm(total, device=DEV, generator=_generator(seed, "order")).to(torch.int32)
    st.table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(width, device=DEV)
    held = at < torch.tensor(used, device=DEV)[:, None]
    st.table[held] = order[: sum(used)]
    st.lens, st.add, st.T = _ints(past), _ints(new), sum(new)
    st.free = torch.cat([order[sum(used):], order[: sum(used)]])
    st.n_free = _ints([total - sum(used)])
    st.longest, st.most = max(new), max(p + n for p, n in zip(past, new))
    if case["kind"] == "plan":
        st.keep = st.lens.clone()
        return st
    H, KV, st.window, _ = SHAPES[case["shape"]]
    x = _normal(seed, "pool", (total, KV, 2, PAGE, HD), 0.8, torch.float32)
    x *= torch.exp2(torch.randint(-2, 3, (total, KV, 2, 1, 1), device=DEV, generator=_generator(seed, "sizes")).float())
    st.scale = _power(_exponent(x.abs().amax((3, 4))))
    st.kv = (x / st.scale[..., None, None]).to(torch.float8_e4m3fn)
    # the pages of this step's tokens are planned already: one plan serves all layers
    st.seqpos = st.lens.clone()
    taken = 0
    rows = []
    for b in range(B):
        need = _pages(past[b] + new[b]) - used[b]
        st.table[b, used[b]: used[b] + need] = order[sum(used) + taken: sum(used) + taken + need]
        taken += need
        pos = torch.arange(past[b], past[b] + new[b], device=DEV)
        rows.append(st.table[b].long()[pos // PAGE] * PAGE + pos % PAGE)
    st.slots = torch.cat(rows).to(torch.int32)
    st.positions = torch.cat([torch.arange(p, p + n, device=DEV) for p, n in zip(past, new)]).to(torch.int32)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st.q_start = _ints(starts)
    st.rows = torch.arange(B, dtype=torch.int32, device=DEV)
    del st.free, st.n_free, st.lens
    if case["kind"] == "write":
        st.k = _normal(seed, "k", (st.T, KV, HD), 1.5)
        st.v = _normal(seed, "v", (st.T, KV, HD), 0.7)
    else:
        st.q = _normal(seed, "q", (st.T, H, HD), 1.2)
    return st


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _exponent(amax):
    """The exponent of a page's scale: the smallest e with amax <= 448 * 2^e (as a float tensor of whole numbers)."""
    mantissa, e = torch.frexp(amax)  # amax = mantissa * 2^e, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(amax > 0, (e - 9 + (mantissa > 0.875)).float(), torch.full_like(amax, LOWEST_EXP)).clamp(min=LOWEST_EXP)


def _power(e):
    """2^e exactly, of whole numbers e that 32-bit numbers have."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _before(counts):
    return torch.cumsum(counts, 0) - counts


def _plain_plan(st):
    """Back to st.keep tokens a request (pages go back on the stack, the last taken on top), then st.add more."""
    B, width = st.table.shape
    N, dev = st.free.shape[0], st.table.device
    j = torch.arange(width, device=dev)
    has, keeps = (st.lens + PAGE - 1) // PAGE, (st.keep + PAGE - 1) // PAGE
    drop = has - keeps
    gone = (j >= keeps[:, None]) & (j < has[:, None])
    place = st.n_free + drop.sum() - 1 - (_before(drop)[:, None] + j - keeps[:, None])
    stack = torch.cat([st.free, st.free[:1]])
    stack.scatter_(0, torch.where(gone, place, N).reshape(-1).long(), st.table.reshape(-1))
    st.free.copy_(stack[:N])
    st.n_free += drop.sum().to(torch.int32)
    st.table.masked_fill_(gone, -1)
    st.lens.copy_(st.keep)

    ends = st.lens + st.add
    need = (ends + PAGE - 1) // PAGE - keeps
    fresh = (j >= keeps[:, None]) & (j < (keeps + need)[:, None])
    place = st.n_free - 1 - (_before(need)[:, None] + j - keeps[:, None])
    st.table.copy_(torch.where(fresh, st.free[place.clamp(0, N - 1).long()], st.table))
    st.n_free -= need.sum().to(torch.int32)
    q_start = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    q_start[1:] = torch.cumsum(st.add, 0)
    i = torch.arange(st.T, dtype=torch.int32, device=dev)
    b = torch.searchsorted(q_start[1:], i, right=True)
    positions = st.lens[b] + i - q_start[b]
    slots = st.table[b, (positions // PAGE).long()] * PAGE + positions % PAGE
    seqpos = st.lens.clone()
    st.lens.copy_(ends)
    return {"positions": positions, "slots": slots, "q_start": q_start, "seqpos": seqpos, "table": st.table, "lens": st.lens, "free": st.free, "n_free": st.n_free}


def _plain_write(st):
    x = torch.stack([st.k, st.v], 2).float()  # [T, KV, 2, HD]
    slots = st.slots.long()
    page, off = slots // PAGE, slots % PAGE
    n, KV = st.kv.shape[:2]
    most = torch.zeros((n, KV, 2), device=x.device).scatter_reduce_(0, page[:, None, None].expand(-1, KV, 2), x.abs().amax(3), "amax")
    # a page that is begun keeps at least its scale; only a request's first page can be one, and its earlier tokens are rounded to the new scale
    first = st.q_start[:-1].long()
    begun, old = page[first], off[first]
    need = _exponent(most)
    grown = torch.where((old > 0)[:, None, None], torch.maximum(torch.frexp(st.scale[begun]).exponent - 1, need[begun]), need[begun])
    raw = st.kv.view(torch.uint8)
    codes = raw[begun]
    again = (codes.view(torch.float8_e4m3fn).float() * (st.scale[begun] / _power(grown))[..., None, None]).to(torch.float8_e4m3fn)
    earlier = torch.arange(PAGE, device=x.device) < old[:, None]
    raw[begun] = torch.where(earlier[:, None, None, :, None], again.view(torch.uint8), codes)
    touched = torch.zeros(n, dtype=torch.bool, device=x.device).scatter_(0, page, True)
    need[begun] = grown
    st.scale.copy_(torch.where(touched[:, None, None], _power(need), st.scale))
    raw[page, :, :, off] = (x / st.scale[page][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return {"kv": st.kv, "scale": st.scale}


def _plain_attend(st):
    """All requests at once, padded to the longest one's queries and to the most pages."""
    T, H, _ = st.q.shape
    KV, B, L = st.kv.shape[1], st.rows.shape[0], _pages(st.most) * PAGE
    pages = st.table[st.rows.long(), : L // PAGE].clamp(min=0).long()
    x = st.kv.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * st.scale[pages][..., None, None]  # [B, pages, KV, 2, PAGE, HD]
    k, v = x.permute(3, 0, 2, 1, 4, 5).reshape(2, B, KV, 1, L, HD)
    i = torch.arange(T, dtype=torch.int32, device=x.device)
    b = torch.searchsorted(st.q_start[1:], i, right=True)
    at = (i - st.q_start[b]).long()
    q = torch.zeros((B, st.longest, H, HD), device=x.device)
    q[b, at] = st.q.float()
    q = q.view(B, st.longest, KV, H // KV, HD).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, k.transpose(3, 4)) * HD ** -0.5  # [B, KV, H / KV, longest, L]
    here = (st.seqpos[:, None] + torch.arange(st.longest, device=x.device))[:, None, None, :, None]
    key = torch.arange(L, device=x.device)
    seen = (key <= here) & (key > here - (st.window or L + 1))
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, st.longest, H, HD)[b, at].to(st.q.dtype).reshape(T, H * HD)


def _plain_score(st):
    x, top = st.logits.float(), st.case["top"]
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    logprob = torch.where(st.targets >= 0, (x.gather(1, st.targets.clamp(min=0)[:, None]) - lse)[:, 0], 0.0)
    entropy = (torch.log(z) - torch.where(e > 0, e * (x - m), 0.0).sum(1, keepdim=True) / z)[:, 0]
    # keys that order like (value, lowest index first), no two of them equal
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    ids = torch.topk((order << 32) + (V - 1 - torch.arange(V, device=x.device)), top, dim=1).indices
    return {"logprob": logprob, "entropy": entropy, "top_ids": ids, "top_logprobs": x.gather(1, ids) - lse}


# ------------------------------------------------------------------------------------------------------------------ the framework's calls
def _own_plan(st):
    from mistral_inference_b200.paged import PageTables
    if not hasattr(st, "tables"):  # the handle that a server keeps over its block tables
        st.tables = PageTables(st.table, st.lens, st.free, st.n_free)
    st.tables.truncate(st.keep)
    plan = st.tables.extend(st.add, st.T, longest=st.longest, most=st.most)
    return {"positions": plan.positions, "slots": plan.slots, "q_start": plan.q_start, "seqpos": plan.seqpos,
            "table": st.table, "lens": st.lens, "free": st.free, "n_free": st.n_free}


def _plan_of(st):
    from mistral_inference_b200.paged import PagePlan
    return PagePlan(table=st.table, rows=st.rows, q_start=st.q_start, seqpos=st.seqpos, positions=st.positions, slots=st.slots, longest=st.longest, most=st.most)


def _own_write(st):
    from mistral_inference_b200.paged import write_pages
    write_pages(st.kv, st.scale, st.k, st.v, _plan_of(st))
    return {"kv": st.kv, "scale": st.scale}


def _own_attend(st):
    from mistral_inference_b200.paged import attend_pages
    return attend_pages(st.q, st.kv, st.scale, _plan_of(st), window=st.window)


def _own_score(st):
    from mistral_inference_b200 import token_scores
    s = token_scores(st.logits, st.targets, top=st.case["top"])
    return {"logprob": s.logprob, "entropy": s.entropy, "top_ids": s.top_ids, "top_logprobs": s.top_logprobs}


def run(st):
    kind = st.case["kind"]
    if own:
        return _own_plan(st) if kind == "plan" else _own_write(st) if kind == "write" else _own_attend(st) if kind == "attend" else _own_score(st)
    return _plain_plan(st) if kind == "plan" else _plain_write(st) if kind == "write" else _plain_attend(st) if kind == "attend" else _plain_score(st)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    if case["kind"] == "score":
        T, V = case["tokens"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * (size * V + 8 + 4 + 4 + 12 * case["top"]), "flops": 6 * T * V}  # maximum, difference, exponential, two sums, product
    new, past, B = _new(case), _past(case), case["batch"]
    T = sum(new)
    fresh = sum(_pages(p + n) - _pages(p) for p, n in zip(past, new))
    if case["kind"] == "plan":
        return {"bytes": 4 * (2 * T + 2 * fresh + 8 * B), "flops": 4 * T}
    H, KV, W, _ = SHAPES[case["shape"]]
    if case["kind"] == "write":
        # each row of 16-bit numbers read, each row of 8-bit numbers written
        return {"bytes": T * KV * 2 * HD * 3, "flops": 4 * T * KV * 2 * HD}
    W = W or 1 << 30
    seen = sum(min(p + i + 1, W) for p, n in zip(past, new) for i in range(n))
    held = sum(min(p + n, W + n - 1) for p, n in zip(past, new))
    return {"bytes": held * KV * 2 * HD + 2 * 2 * T * H * HD, "flops": 4 * H * HD * seen}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def _e4m3(x):
    """The e4m3 number next to x (64 bits, |x| <= 448), ties to the even one: steps of 2^(binade - 3), 2^-9 below 2^-6."""
    binade = _ceil_power(x.abs().clamp(min=2.0 ** -6))
    step = torch.where(binade > x.abs().clamp(min=2.0 ** -6), binade / 2, binade) / 8
    return torch.round(x / step) * step


def _ceil_power(x):
    """The smallest power of two that is not below x > 0, in 64 bits."""
    e = torch.floor(torch.log2(x)).long()  # (may be one off next to a power)
    power = lambda n: ((n + 1023) << 52).view(torch.float64)  # noqa: E731
    e -= (power(e) > x).long()
    return power(e + (power(e) < x).long())


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    st = prepare(case, seed)
    if case["kind"] == "score":
        out = {"logprob": [], "entropy": [], "top_ids": None, "top_logprobs": []}
        for row, target in zip(st.logits, st.targets.tolist()):
            lp = torch.log_softmax(row.double(), 0)
            p = lp.exp()
            out["logprob"].append(lp[target] if target >= 0 else lp.new_zeros(()))
            out["entropy"].append(-(p * lp)[p > 0].sum())
            out["top_logprobs"].append(lp.sort(descending=True).values[: case["top"]])
        return {k: torch.stack(v) if v is not None else None for k, v in out.items()}
    starts = st.q_start.tolist()
    if case["kind"] == "write":
        kv, scale = st.kv.double(), st.scale.double()
        for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
            t = lo
            while t < hi:  # page by page
                slot = int(st.slots[t])
                page, off = slot // PAGE, slot % PAGE
                n = min(hi - t, PAGE - off)
                x = torch.stack([st.k[t:t + n], st.v[t:t + n]], 2).double().permute(1, 2, 0, 3)  # [KV, 2, n, HD]
                size = _ceil_power((x.abs().amax((2, 3)) / E4M3_MAX).clamp(min=2.0 ** LOWEST_EXP))
                if off:
                    size = torch.maximum(size, scale[page])
                    kv[page, :, :, :off] = _e4m3(kv[page, :, :, :off] * (scale[page] / size)[..., None, None])
                scale[page] = size
                kv[page, :, :, off:off + n] = _e4m3(x / scale[page][..., None, None])
                t += n
        return {"kv": kv, "scale": scale}
    H, KV = st.q.shape[1], st.kv.shape[1]
    out = torch.empty(st.T, H, HD, dtype=torch.float64, device=DEV)
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        past = int(st.seqpos[b])
        keys = past + hi - lo
        pages = st.table[b, : _pages(keys)].long()
        x = (st.kv.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * st.scale[pages].double()[..., None, None]).permute(2, 1, 0, 3, 4).reshape(2, KV, -1, HD)[:, :, :keys]
        for g in range(KV):
            heads = slice(g * (H // KV), (g + 1) * (H // KV))
            s = torch.einsum("thd,kd->htk", st.q[lo:hi, heads].double(), x[0, g]) / math.sqrt(HD)
            gap = torch.arange(past, keys, device=DEV)[:, None] - torch.arange(keys, device=DEV)
            s = s.masked_fill((gap < 0) | (gap >= (st.window or keys + 1)), -math.inf)
            out[lo:hi, heads] = torch.einsum("htk,kd->thd", torch.softmax(s, -1), x[1, g])
    return out.reshape(st.T, H * HD)
