"""The Transformer with 8-bit weights: the whole path through forward and generate, its Linears held against 64-bit restatements of the same operators."""
import json

import pytest
import safetensors.torch
import torch

import mistral_inference_b200 as mi
import synth
from mistral_inference_b200 import _abi_rows8, rows8
from mistral_inference_b200._abi import Mb200Error
from mistral_inference_b200.main import main
from mistral_inference_b200.rows8 import Rows8
from mistral_inference_b200.transformer import Transformer

from . import rows8_util as U

pytestmark = pytest.mark.gpu


def model_of(name="tiny", max_batch=4, seed=1, head=None, **over):
    p = synth.shape(name, **over)
    args = mi.TransformerArgs.from_dict(dict(p))
    args.max_batch_size = max_batch
    m = Transformer.empty(args, "cuda", torch.bfloat16)
    m.load_state_dict(synth.synth_state_dict(p, seed, torch.bfloat16, "cuda"))
    if head is not None:
        m.quantise_weights(head=head)
    return m.eval(), p


def plain_rows(y):
    codes, scales = U.quantised(y.float())
    return Rows8(codes, scales.view(torch.float8_e8m0fnu), y.shape[1])


def values(x):
    return U.numbers(x.codes, x.scales, x.cols)


def plain_norm(x, weight, eps, add=None):
    h = x if add is None else (x.double() + add.double()).to(x.dtype)
    return plain_rows(h.double() / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + eps) * weight.double()), h


def plain_multiply(x, w, dtype=torch.bfloat16, out=None):
    y = values(x) @ values(w).t()
    return y.to(dtype) if out is None else out.copy_(y)


def plain_gate(x, w):
    y = values(x) @ values(w).t()
    return plain_rows(y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2])


@pytest.fixture
def plain_linears(monkeypatch):
    """The Linears by the restatements: what the model computes then differs by roundings alone."""
    own = {n: getattr(rows8, n) for n in ("quantise_rows", "norm_rows", "multiply_rows", "gate_rows")}

    def use(on):
        for n, f in (("quantise_rows", plain_rows), ("norm_rows", plain_norm), ("multiply_rows", plain_multiply), ("gate_rows", plain_gate)):
            monkeypatch.setattr(rows8, n, f if on else own[n])
    monkeypatch.setenv("MB200_DECODE_GRAPH", "0")
    return use


@pytest.mark.parametrize("kv_cache", ["ring", "pages"])
@pytest.mark.parametrize("head", [False, True])
@pytest.mark.parametrize("over", [{}, {"sliding_window": 50}, {"hidden_dim": 704, "vocab_size": 1003}])
def test_forward(over, head, kv_cache, plain_linears):
    """Sums of another order round otherwise here and there: a 16-bit result by 2^-8 of itself (some one in ten thousand), a code by up to 2^-3 of itself (one in a million).  One such entry among
    the 256 and more of a row moves what is computed of it by at most 2^-3 / sqrt(256) = 2^-7 of its spread, and there are a few of them behind a token's logits.  A mistake in rows or
    scales moves them by as much as they are."""
    if over.get("vocab_size") == 1003 and not head:
        over = {**over, "vocab_size": 1002}  # (the 16-bit head takes even vocabularies only)
    m, p = model_of(head=head, **over)
    g = torch.Generator().manual_seed(3)
    steps = [[70, 3, 129], [1, 1, 1], [20, 64, 1], [1, 1, 1], [1, 1, 1]]
    ids = [torch.randint(0, p["vocab_size"], (sum(s),), generator=g).cuda() for s in steps]
    outs = []
    for plain in (False, True):
        plain_linears(plain)
        cache = m.make_cache(3, 300, kv_cache=kv_cache)
        outs.append([m.forward(x, s, cache) for x, s in zip(ids, steps)] + [m.forward(ids[0][:9], [9])])
    for got, want in zip(*outs):
        assert torch.isfinite(got).all() and (got - want).abs().max() <= 2.0 ** -4 * want.std() and (got - want).std() <= 2.0 ** -6 * want.std(), ((got - want).abs().max(), want.std())


def test_weights_of_8_bits_stay_near_those_of_16():
    """A weight and an activation of 4 significant bits: each Linear's result is off by some 2^-5.3 sqrt(2) of its spread with either sign, fourteen Linears one behind another or side by
    side.  A mistake moves logits by as much as they are."""
    out = []
    for head in (None, False, True):
        m, p = model_of(head=head)
        ids = torch.randint(0, p["vocab_size"], (120,), generator=torch.Generator().manual_seed(5)).cuda()
        out.append(m.forward(ids, [60, 60], m.make_cache(2, 200)).float())
    assert (out[1] - out[0]).std() <= 2.0 ** -2 * out[0].std() and (out[2] - out[0]).std() <= 2.0 ** -2 * out[0].std()
    assert not torch.equal(out[0], out[1]) and not torch.equal(out[1], out[2])


@pytest.mark.parametrize("kv_cache", ["ring", "pages"])
@pytest.mark.parametrize("B", [1, 3])
def test_decode_steps_replayed_are_decode_steps_run(B, kv_cache, monkeypatch):
    m, p = model_of(head=True)
    outs = []
    for graph in ("1", "0"):
        monkeypatch.setenv("MB200_DECODE_GRAPH", graph)
        cache = m.make_cache(B, 200, kv_cache=kv_cache)
        x = m.forward((torch.arange(60 * B) % p["vocab_size"]).cuda(), [60] * B, cache)
        nxt = torch.arange(5, 5 + B, device="cuda")
        outs.append((x, [m.forward(nxt + i, [1] * B, cache).clone() for i in range(8)]))
    assert torch.equal(outs[0][0], outs[1][0])
    for a, b in zip(outs[0][1], outs[1][1]):
        assert torch.equal(a, b)


def test_a_cache_that_was_decoded_with_16_bits_goes_on_with_8():
    """Its captured step read matrices that are gone."""
    a, p = model_of()
    b, _ = model_of(head=False)
    cache = a.make_cache(2, 100)
    ids = (torch.arange(40) % p["vocab_size"]).cuda()
    a.forward(ids, [20, 20], cache)
    nxt = torch.tensor([5, 6], device="cuda")
    for i in range(4):
        a.forward(nxt, [1, 1], cache)
    other = b.make_cache(2, 100)
    for x, y in zip(cache.cache_k + cache.cache_v if isinstance(cache.cache_k, list) else list(cache.cache_k.values()) + list(cache.cache_v.values()),
                    other.cache_k + other.cache_v if isinstance(other.cache_k, list) else list(other.cache_k.values()) + list(other.cache_v.values())):
        y.copy_(x)
    other.update_seqlens([24, 24]) if other.kv_seqlens is not None else (other.init_kvseqlens(2), other.update_seqlens([24, 24]))
    a.quantise_weights()
    for i in range(4):
        assert torch.equal(a.forward(nxt + i, [1, 1], cache), b.forward(nxt + i, [1, 1], other))


@pytest.mark.parametrize("kv_cache", ["ring", "pages"])
def test_generate(kv_cache):
    m, p = model_of(head=True)
    prompts = [synth.synth_prompt(n, p["vocab_size"], 2 + i) for i, n in enumerate((40, 33, 37))]
    toks, lps, details = mi.generate(prompts, m, max_tokens=6, temperature=0.0, chunk_size=16, kv_cache=kv_cache, alternatives=3)
    for t, lp, d in zip(toks, lps, details):
        assert [x.top_ids[0] for x in d[-6:]] == t and [x.top_logprobs[0] for x in d[-6:]] == lp[-6:]
    again, lps2 = mi.generate(prompts, m, max_tokens=6, temperature=0.0, chunk_size=16, kv_cache=kv_cache)
    assert again == toks and all(abs(a - b) <= 1e-4 for x, y in zip(lps, lps2) for a, b in zip(x, y))
    # a prompt with the generated tokens behind it scores them as they were picked (prompts and steps sum in another order: see test_forward)
    _, full = mi.generate([q + t for q, t in zip(prompts, toks)], m, max_tokens=0, temperature=0.0, chunk_size=16, kv_cache="ring")
    if kv_cache == "ring":
        assert max(abs(a - b) for x, y in zip(lps, full) for a, b in zip(x, y)) <= 0.1


def test_the_16_bit_matrices_are_given_up():
    torch.cuda.synchronize()
    m, p = model_of(dim=1024, hidden_dim=4096, n_heads=8)
    before = torch.cuda.memory_allocated()
    linears = sum(w.numel() for b in m.layers.values() for w in (b.attention.wqkv, b.attention.wo_weight, b.feed_forward.w13, b.feed_forward.w2_weight))
    m.quantise_weights()
    kept = [r for b in m.layers.values() for r in (b.attention.wqkv8, b.attention.wo8, b.feed_forward.w13_8, b.feed_forward.w2_8)]
    assert all(r.fixed for r in kept)
    assert all(w.numel() == 0 for b in m.layers.values() for w in (b.attention.wqkv, b.attention.wo_weight, b.feed_forward.w13, b.feed_forward.w2_weight))
    storages = {s.data_ptr(): s.nbytes() for r in kept for s in (r.codes.untyped_storage(), r.scales.untyped_storage())}  # (codes and scales share one)
    assert sum(storages.values()) <= linears * (1 + 1 / 64)
    # (a block that the allocator has left over from others may be up to 1 MiB larger than what it is asked for, and counts as a whole: one for each matrix, or its codes' and its scales')
    assert before - torch.cuda.memory_allocated() >= linears * 2 - linears * (1 + 1 / 64) - 2 * len(kept) * (1 << 20)
    for call in (m.quantise_weights, m.state_dict, lambda: m.load_state_dict({}), lambda: m._load_lora_state_dict({"lora": torch.zeros(1, dtype=torch.bfloat16)})):
        with pytest.raises(Mb200Error, match="8 bits"):
            call()


def test_mixtures_are_refused():
    m, _ = model_of("tiny-moe")
    with pytest.raises(Mb200Error, match="dense"):
        m.quantise_weights()


def test_from_folder_and_command_line(tmp_path, capsys):
    p = synth.shape("tiny")
    safetensors.torch.save_file({k: v.contiguous() for k, v in synth.synth_state_dict(p, 1).items()}, str(tmp_path / "consolidated.safetensors"))
    (tmp_path / "params.json").write_text(json.dumps(p))
    a = Transformer.from_folder(tmp_path, max_batch_size=2, weights="e4m3")
    b, _ = model_of(max_batch=2, head=False)
    ids = (torch.arange(50) % p["vocab_size"]).cuda()
    assert a.weights8 and torch.equal(a.forward(ids, [30, 20], a.make_cache(2, 60)), b.forward(ids, [30, 20], b.make_cache(2, 60)))
    with pytest.raises(ValueError):
        Transformer.from_folder(tmp_path, weights="int8")
    toks, _ = mi.generate([[5, 17, 3]], Transformer.from_folder(tmp_path, weights="e4m3"), max_tokens=4, temperature=0.0)
    assert main(["generate", str(tmp_path), "--prompt", "5 17 3", "--max-tokens", "4", "--weights", "e4m3"]) == 0
    assert capsys.readouterr().out.split() == [str(t) for t in toks[0]]


@pytest.mark.parametrize("T,H,KV", [(1, 4, 2), (7, 32, 8), (300, 6, 1)])
def test_rotation(T, H, KV):
    """Bit for bit what the 16-bit path's product does behind its rounding: the reference's complex product in 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, (H + 2 * KV) * 128, device="cuda", generator=g).bfloat16()
    angle = torch.rand(500, 64, device="cuda", generator=g) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], 2).contiguous()
    positions = torch.randint(0, 500, (T,), device="cuda", generator=g).int()
    x = torch.view_as_complex(qkv[:, : (H + KV) * 128].float().view(T, H + KV, 64, 2))
    want = torch.view_as_real(x.cpu() * torch.view_as_complex(rope).cpu()[positions.cpu().long()][:, None]).flatten(2).bfloat16().cuda()
    rows = torch.randperm(T + 5, device="cuda", generator=g)[:T].int()
    if T > 1:
        rows[T // 2] = -1
    for at in (None, rows):
        n = T if at is None else T + 5
        q = torch.zeros(T, H * 128, device="cuda", dtype=torch.bfloat16)
        k, v = torch.full((2, n, KV * 128), 7.0, device="cuda", dtype=torch.bfloat16)
        _abi_rows8.rotate(qkv, rope, positions, at, q, k, v, H, KV)
        assert torch.equal(q.view(T, H, 128), want[:, :H])
        place = torch.arange(T, device="cuda") if at is None else at.long()
        there = place >= 0
        assert torch.equal(k[place[there]].view(-1, KV, 128), want[there][:, H:]) and torch.equal(v[place[there]], qkv[there][:, (H + KV) * 128:])
        rest = torch.ones(n, dtype=torch.bool, device="cuda")
        rest[place[there]] = False
        assert (k[rest] == 7).all() and (v[rest] == 7).all()


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("head", [None, True])
def test_a_model_that_was_moved_goes_on(B, head):
    """To the host and back between the steps of a cache: what was captured before reads memory that is gone."""
    m, p = model_of(head=head)
    still, _ = model_of(head=head)
    caches = [m.make_cache(B, 100), still.make_cache(B, 100)]
    ids = (torch.arange(20 * B) % p["vocab_size"]).cuda()
    nxt = torch.arange(5, 5 + B, device="cuda")
    for model, cache in zip((m, still), caches):
        model.forward(ids, [20] * B, cache)
    for i in range(9):
        if i == 4:
            m.cpu()
            if head:
                with pytest.raises(Mb200Error):
                    m.forward(nxt, [1] * B)
            taken = [torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda") for n in (1 << 20, 1 << 21, 1 << 22)]  # where the matrices were
            m.cuda()
            del taken
        a, b = (model.forward(nxt + i, [1] * B, cache) for model, cache in zip((m, still), caches))
        assert torch.equal(a, b), i


def test_the_last_addition_is_the_8_bit_heads(monkeypatch):
    """Every addition to the stream is made by the norm behind it, the head's norm too; the same bits as an addition ahead of it, in every call that has logits or scores."""
    m, p = model_of(head=True)
    own, adds = rows8.norm_rows, []
    ids = (torch.arange(300) * 7 % p["vocab_size"]).cuda()
    targets = ids.roll(-1)
    nxt = torch.tensor([5, 6], device="cuda")

    def run():
        adds.clear()
        cache, other = m.make_cache(2, 400), m.make_cache(2, 400)
        first = m.forward(ids, [170, 130], cache)
        step = m.forward(nxt, [1, 1], cache).clone()
        scored = m.forward_logprobs(ids, [170, 130], None, targets)
        scores, last = m.forward_scores(ids, [170, 130], other, targets, 3)
        return [first, step, *scored, scores.logprob, scores.entropy, scores.top_ids, scores.top_logprobs, last, m.forward_partial(ids[:9], [9])]

    def together(x, weight, eps, add=None):
        adds.append(add is not None)
        return own(x, weight, eps, add=add)

    def ahead(x, weight, eps, add=None):
        h = x if add is None else x + add
        return own(h, weight, eps)[0], h
    monkeypatch.setattr(rows8, "norm_rows", together)
    got = run()
    layers = [False] + [True] * (2 * p["n_layers"] - 1)
    assert adds == (layers + [True]) * 4 + layers  # (forward_partial's last norm is in 16 bits)
    monkeypatch.setattr(rows8, "norm_rows", ahead)
    for a, b in zip(got, run()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kv_cache", ["ring", "pages"])
def test_decode_steps_of_many_sequences(kv_cache, monkeypatch):
    """More sequences than the products for a few tokens take: captured steps whose products have parts in memory of their own, of two caches in turn."""
    m, p = model_of(head=True, max_batch=150, dim=512, n_heads=4, hidden_dim=4096)
    prompts = [(torch.arange(150 * 3) * k % p["vocab_size"]).cuda() for k in (7, 11)]
    nxt = torch.arange(150, device="cuda")
    outs = {}
    for graph in ("0", "1"):
        monkeypatch.setenv("MB200_DECODE_GRAPH", graph)
        caches = [m.make_cache(150, 40, kv_cache=kv_cache) for _ in range(2)]
        outs[graph] = [[m.forward(ids, [3] * 150, c)] for ids, c in zip(prompts, caches)]
        for i in range(5):
            for j, c in enumerate(caches):
                outs[graph][j].append(m.forward((nxt + i + j) % p["vocab_size"], [1] * 150, c).clone())
    for a, b in zip(outs["0"], outs["1"]):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
