"""The Transformer on 8-bit pages: the whole path through forward and generate, its attention held against 64 bits over the same pages."""
import re

import pytest
import torch

import mistral_inference_b200 as mi
import synth
from mistral_inference_b200 import paged
from mistral_inference_b200.transformer import Transformer

from . import paged_util as U
from .util import logit_tol

pytestmark = pytest.mark.gpu


def model_of(name="tiny", max_batch=4, seed=1, **over):
    p = synth.shape(name, **over)
    args = mi.TransformerArgs.from_dict(dict(p))
    args.max_batch_size = max_batch
    m = Transformer.empty(args, "cuda", torch.bfloat16)
    m.load_state_dict(synth.synth_state_dict(p, seed, torch.bfloat16, "cuda"))
    return m.eval(), p


@pytest.fixture
def plain_attention(monkeypatch):
    """Attention over pages by the 64-bit restatement: what the model computes then differs by roundings alone."""
    def attend(q, kv, scale, plan, window=0, softmax_scale=None, out=None):
        q_start, table = plan.q_start.tolist(), plan.table.tolist()
        o, _ = U.attend_ref(q.cpu().view(q.shape[0], -1, 128), kv.cpu().double(), scale.cpu(), table, plan.rows.tolist(), q_start, plan.seqpos.tolist(), window, softmax_scale)
        return out.copy_(o.reshape(out.shape).to(out))
    def use(on):
        monkeypatch.setattr(paged, "attend_pages", attend if on else mi.attend_pages)
    monkeypatch.setenv("MB200_DECODE_GRAPH", "0")
    return use


# Two correct attentions differ by a bf16 rounding of their outputs here and there (and by the weights' 2^-8, see attend_tolerance); as for prompts over 16-bit rings, logits then
# differ by two bf16 steps at the scale of the largest, three with the weights' roundings on both sides.
ULPS = 3


@pytest.mark.parametrize("name,over", [("tiny", {}), ("tiny", {"sliding_window": 50}), ("tiny", {"sliding_window": [24, None], "n_layers": 4}), ("tiny-moe", {})])
def test_forward_on_pages(name, over, plain_attention):
    m, p = model_of(name, **over)
    g = torch.Generator().manual_seed(3)
    steps = [[70, 3, 129], [1, 1, 1], [20, 64, 1], [1, 1, 1], [1, 1, 1]]
    ids = [torch.randint(0, p["vocab_size"], (sum(s),), generator=g).cuda() for s in steps]
    outs = []
    for plain in (False, True):
        plain_attention(plain)
        cache = m.make_cache(3, 300, kv_cache="pages")
        outs.append([m.forward(x, s, cache) for x, s in zip(ids, steps)])
        assert cache.kv_seqlens.tolist() == [sum(s[b] for s in steps) for b in range(3)]
    for got, want in zip(*outs):
        assert torch.isfinite(got).all()
        if name == "tiny":  # (a router's choice between two nearly equal experts may fall otherwise)
            assert (got - want).abs().max() <= logit_tol(want, ULPS), (got - want).abs().max()


def test_first_prompts_are_those_of_rings():
    """A batch's first tokens attend over their own 16-bit rows, whatever the cache."""
    m, p = model_of()
    ids = torch.arange(200).cuda() % p["vocab_size"]
    a = m.forward(ids, [130, 70], m.make_cache(2, 200, kv_cache="pages"))
    b = m.forward(ids, [130, 70], m.make_cache(2, 200))
    assert torch.equal(a, b)


def test_pages_stay_near_rings():
    """Keys and values of 4 significant bits instead of 8: logits move, but by a few hundredths of their spread.  (Each number is off by at most 2^-4 of itself, some 2^-5.5 on
    average with either sign; sums over 128 dimensions and 60 keys average them: 2^-5.5 / sqrt(8) of a score's spread, times a few layers.  A mistake in rows or scales moves them by as much
    as they are.)"""
    m, p = model_of()
    g = torch.Generator().manual_seed(5)
    prompt, nxt = torch.randint(0, p["vocab_size"], (120,), generator=g).cuda(), torch.randint(0, p["vocab_size"], (2,), generator=g).cuda()
    out = []
    for kind in ("pages", "ring"):
        c = m.make_cache(2, 200, kv_cache=kind)
        m.forward(prompt, [60, 60], c)
        out.append(m.forward(nxt, [1, 1], c).float())
    assert (out[0] - out[1]).std() <= 2.0 ** -3 * out[1].std()


def test_decode_steps_replayed_are_decode_steps_run(monkeypatch):
    m, p = model_of()
    outs = []
    for graph in ("1", "0"):
        monkeypatch.setenv("MB200_DECODE_GRAPH", graph)
        cache = m.make_cache(3, 200, kv_cache="pages")
        x = m.forward((torch.arange(140) % p["vocab_size"]).cuda(), [60, 17, 63], cache)
        nxt = torch.tensor([5, 6, 7], device="cuda")
        got = []
        for i in range(8):  # a page boundary inside
            got.append(m.forward(nxt + i, [1, 1, 1], cache).clone())
        cache.update_seqlens([-3, -1, 0])  # drafted tokens taken back
        for i in range(4):
            got.append(m.forward(nxt + i, [1, 1, 1], cache).clone())
        got.append(m.forward(torch.arange(12).cuda(), [4, 4, 4], cache))
        got.append(m.forward(nxt, [1, 1, 1], cache).clone())
        outs.append((x, got, cache.tables.lens.tolist(), cache.ledger.lens))
    assert outs[0][2:] == outs[1][2:] and outs[0][2] == [60 + 8 - 3 + 9, 17 + 8 - 1 + 9, 63 + 8 + 9]
    for a, b in zip(outs[0][1], outs[1][1]):
        assert torch.equal(a, b)


def test_one_request_alone_in_a_batch_of_one():
    """Batch 1 on rings is one persistent kernel; on pages it is the layers' own."""
    m, p = model_of(max_batch=1)
    cache = m.make_cache(1, 100, kv_cache="pages")
    m.forward(torch.arange(50).cuda(), [50], cache)
    a = [m.forward(torch.tensor([i], device="cuda"), [1], cache).clone() for i in range(4)]
    again = m.make_cache(1, 100, kv_cache="pages")
    m.forward(torch.arange(50).cuda(), [50], again)
    b = m.forward(torch.tensor([0, 1, 2, 3], device="cuda"), [4], again)
    for i in range(4):  # steps of one token, and the same tokens at once (written before any of them attends)
        assert (a[i][0] - b[i]).abs().max() <= logit_tol(b, ULPS)


def test_requests_come_and_go():
    """A running batch: one request ends, another takes its row and pages; the others do not notice."""
    m, p = model_of(max_batch=3)
    V = p["vocab_size"]
    cache = m.make_cache(3, 300, kv_cache="pages", n_pages=8)
    first = [(torch.arange(n) * 7 % V).cuda() for n in (100, 65, 30)]
    m.forward(torch.cat(first), [100, 65, 30], cache)
    with pytest.raises(ValueError, match="pages"):
        m.forward(torch.zeros(250, dtype=torch.long, device="cuda"), [50, 200, 0], cache)
    step = m.forward(torch.tensor([1, 2, 3], device="cuda"), [1, 1, 1], cache).clone()
    cache.retire([1])
    assert cache.rows == [0, 2] and cache.kv_seqlens.tolist() == [101, 31] and int(cache.tables.n_free) == cache.ledger.free_pages == 5
    assert cache.admit(1) == [2] and cache.rows == [0, 2, 1]
    new = (torch.arange(150) * 3 % V).cuda()
    m.forward(new, [0, 0, 150], cache)  # a prompt beside requests that bring nothing
    got = m.forward(torch.tensor([4, 5, 6], device="cuda"), [1, 1, 1], cache).clone()
    assert cache.tables.lens.tolist() == [102, 151, 32] and step.shape == (3, V)
    # the same requests, never in company of the one that ended
    other = m.make_cache(3, 300, kv_cache="pages")
    m.forward(torch.cat([first[0], first[2]]), [100, 30], other)
    m.forward(torch.tensor([1, 3], device="cuda"), [1, 1], other)
    other.admit(1)
    m.forward(new, [0, 0, 150], other)
    want = m.forward(torch.tensor([4, 5, 6], device="cuda"), [1, 1, 1], other)
    assert (got - want).abs().max() <= logit_tol(want, ULPS)


def test_a_first_prompt_beside_requests_that_bring_nothing():
    m, p = model_of(max_batch=3)
    V = p["vocab_size"]
    prompt = [(torch.arange(n) * 7 % V).cuda() for n in (90, 33)]
    a, b = m.make_cache(3, 300, kv_cache="pages"), m.make_cache(3, 300, kv_cache="pages")
    got = m.forward(prompt[0], [0, 90, 0], a)
    got = torch.cat([got, m.forward(prompt[1], [33, 0, 0], a)])
    step = m.forward(torch.tensor([4, 5], device="cuda"), [1, 1, 0], a)
    want = m.forward(prompt[0], [90], b)
    b.admit(1)
    want = torch.cat([want, m.forward(prompt[1], [0, 33], b)])
    assert (got[:90] - want[:90]).abs().max() <= logit_tol(want, ULPS) and (got[90:] - want[90:]).abs().max() <= logit_tol(want, ULPS)
    want = m.forward(torch.tensor([5, 4], device="cuda"), [1, 1], b)
    assert (step - want[[1, 0]]).abs().max() <= logit_tol(want, ULPS)
    with pytest.raises(AssertionError, match="brings a token"):
        m.forward_scores(prompt[0], [0, 90, 0], a, torch.zeros(90, dtype=torch.long, device="cuda"), 3)


def test_a_step_that_fails_leaves_no_tokens_behind(monkeypatch):
    m, p = model_of(max_batch=2)
    cache = m.make_cache(2, 100, kv_cache="pages")
    m.forward(torch.arange(80).cuda(), [40, 40], cache)
    layer = m.layers["1"]
    def broken(*a):
        raise RuntimeError("lost")
    with monkeypatch.context() as mp:
        mp.setattr(type(layer), "forward", broken)
        with pytest.raises(RuntimeError, match="lost"):
            m.forward(torch.arange(60).cuda(), [30, 30], cache)
    assert cache.kv_seqlens.tolist() == [40, 40] and cache.tables.lens.tolist() == [70, 70]
    m.forward(torch.arange(2).cuda(), [1, 1], cache)
    assert cache.tables.lens.tolist() == [41, 41] and int(cache.tables.n_free) == cache.ledger.free_pages


@pytest.mark.parametrize("kv_cache,temperature", [("ring", 0.0), ("pages", 0.0), ("pages", 0.7)])
def test_generate_reports_alternatives(kv_cache, temperature):
    m, p = model_of(max_batch=2)
    prompts = [[1 + i for i in range(40)], [9, 8, 7, 6, 5]]
    kw = dict(max_tokens=7, temperature=temperature, chunk_size=None, kv_cache=kv_cache)
    torch.manual_seed(1)
    tokens, lps, details = mi.generate(prompts, m, alternatives=4, **kw)
    torch.manual_seed(1)
    tokens2, lps2 = mi.generate(prompts, m, **kw)
    assert tokens == tokens2
    for b in range(2):
        assert len(lps[b]) == len(details[b]) == len(prompts[b]) - 1 + 7
        # 2^-16: sums over the vocabulary in two orders
        assert max(abs(x - y) for x, y in zip(lps[b], lps2[b])) <= 2.0 ** -14 * 16
        chosen = prompts[b][1:] + tokens[b]
        for t, lp, d in zip(chosen, lps[b], details[b]):
            assert len(d.top_ids) == 4 and d.top_logprobs == sorted(d.top_logprobs, reverse=True) and d.entropy >= 0
            assert d.top_ids.index(t) >= 0 and abs(d.top_logprobs[d.top_ids.index(t)] - lp) < 1e-5 if t in d.top_ids else lp <= d.top_logprobs[-1] + 1e-5
        if temperature == 0.0:
            assert [d.top_ids[0] for d in details[b][len(prompts[b]) - 1:]] == tokens[b]


def test_generate_on_pages_takes_portions_and_stops():
    m, p = model_of(max_batch=2, sliding_window=64)
    prompts = [[(3 * i) % p["vocab_size"] for i in range(200)], [(5 * i + 1) % p["vocab_size"] for i in range(190)]]
    whole, _ = mi.generate(prompts, m, max_tokens=5, temperature=0.0, kv_cache="pages")
    parts, lps = mi.generate(prompts, m, max_tokens=5, temperature=0.0, kv_cache="pages", chunk_size=70)
    assert len(whole[0]) == len(parts[0]) == 5 and len(lps[1]) == 189 + 5
    stopped, _ = mi.generate(prompts[:1], m, max_tokens=5, temperature=0.0, kv_cache="pages", eos_id=mi.generate(prompts[:1], m, max_tokens=5, temperature=0.0, kv_cache="pages")[0][0][2])
    assert len(stopped[0]) <= 2


def test_command_line(tmp_path, capsys):
    from mistral_inference_b200.main import main
    synth.write_model_folder(tmp_path, synth.shape("tiny"), 2)
    assert main(["generate", str(tmp_path), "--prompt", "5 17 3", "--prompt", "1 2 3 4", "--max-tokens", "3", "--kv-cache", "pages", "--alternatives", "2"]) == 0
    lines = capsys.readouterr().out.strip().split("\n")
    assert len(lines) == 2 * (1 + 3) and "entropy" in lines[1] and lines[1].split()[0] == lines[0].split()[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layered_decoders_report_alternatives(tmp_path, dtype):
    from .test_gpu_fesenex import _model
    m, cfg, _ = _model(tmp_path, "mixed", dtype)
    m.args.max_batch_size = 2
    prompts = [[1, 2, 3, 4, 5], [7, 8, 9]]
    tokens, lps, details = mi.generate(prompts, m, max_tokens=4, temperature=0.0, alternatives=3)
    tokens2, lps2 = mi.generate(prompts, m, max_tokens=4, temperature=0.0)
    assert tokens == tokens2
    for b in range(2):
        assert [d.top_ids[0] for d in details[b][len(prompts[b]) - 1:]] == tokens[b] and max(abs(x - y) for x, y in zip(lps[b], lps2[b])) <= 2.0 ** -10
    with pytest.raises(ValueError, match="rings"):
        mi.generate(prompts, m, max_tokens=1, temperature=0.0, kv_cache="pages")


@pytest.mark.parametrize("where", ["warm-up", "capture", "replay"])
def test_a_decode_step_that_fails_leaves_no_tokens_behind(monkeypatch, where):
    """A layer raises in a single-token step (run eagerly, or captured), or the replay does before anything is enqueued: the steps after it are those of a cache that never failed."""
    monkeypatch.setenv("MB200_DECODE_GRAPH", "1")
    m, p = model_of(max_batch=2)
    runs = []
    for fails in (False, True):
        cache = m.make_cache(2, 200, kv_cache="pages")
        m.forward(torch.arange(126).cuda(), [63, 63], cache)  # the next token but one of each begins a page
        steps = 0
        def step():
            nonlocal steps
            steps += 1
            return m.forward(torch.tensor([steps, steps + 1], device="cuda"), [1, 1], cache).clone()
        got = [step() for _ in range({"warm-up": 0, "capture": 1, "replay": 2}[where])]
        if fails:
            def broken(*a):
                raise RuntimeError("lost")
            with monkeypatch.context() as mp:
                if where == "replay":
                    mp.setattr(torch.cuda.CUDAGraph, "replay", broken)
                else:
                    mp.setattr(type(m.layers["1"]), "forward", broken)
                with pytest.raises(RuntimeError, match="lost"):
                    m.forward(torch.tensor([steps + 1, steps + 2], device="cuda"), [1, 1], cache)
            assert cache.kv_seqlens.tolist() == [63 + steps] * 2
        got += [step() for _ in range(5)]
        runs.append((got, cache.tables.lens.tolist(), cache.ledger.lens, int(cache.tables.n_free)))
    assert runs[0][1:] == runs[1][1:] and runs[0][1] == runs[0][2]
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a, b)


def test_a_decode_step_captured_without_tokens_sees_those_that_come():
    """Requests that have given all their tokens back when the step is captured: its replays attend over what they have by then."""
    m, p = model_of(max_batch=2)
    steps = [torch.tensor(t, device="cuda") for t in ([5, 6], [7, 8], [9, 1], [2, 3])]
    cache = m.make_cache(2, 100, kv_cache="pages")
    cache.admit(2)
    m.decode_static(steps[0], cache)
    cache.update_seqlens([-1, -1])
    got = [m.decode_static(t, cache).clone() for t in steps]
    other = m.make_cache(2, 100, kv_cache="pages")
    other.admit(2)
    for i, t in enumerate(steps):
        other.__dict__.pop("_mb200_decode_states", None)  # run, not captured
        assert torch.equal(got[i], m.decode_static(t, other)), i
    # the same tokens without the second: what came before a token matters
    other.update_seqlens([-3, -3])
    assert other.kv_seqlens.tolist() == [1, 1] and not torch.equal(got[2], m.decode_static(steps[2], other))


def test_forward_of_a_mixture_on_pages(plain_attention):
    """test_forward_on_pages for a model whose experts are all alike: whichever the router takes between two that are nearly equal, the numbers are the same."""
    p = synth.shape("tiny-moe")
    args = mi.TransformerArgs.from_dict(dict(p))
    args.max_batch_size = 3
    sd = synth.synth_state_dict(p, 1, torch.bfloat16, "cuda")
    alike = {k: sd[re.sub(r"experts\.\d+\.", "experts.0.", k)] for k in sd}
    assert any(alike[k] is not sd[k] for k in sd)
    m = Transformer.empty(args, "cuda", torch.bfloat16)
    m.load_state_dict(alike)
    m.eval()
    g = torch.Generator().manual_seed(3)
    steps = [[70, 3, 129], [1, 1, 1], [20, 64, 1], [1, 1, 1]]
    ids = [torch.randint(0, p["vocab_size"], (sum(s),), generator=g).cuda() for s in steps]
    outs = []
    for plain in (False, True):
        plain_attention(plain)
        cache = m.make_cache(3, 300, kv_cache="pages")
        outs.append([m.forward(x, s, cache) for x, s in zip(ids, steps)])
    for got, want in zip(*outs):
        assert (got - want).abs().max() <= logit_tol(want, ULPS), (got - want).abs().max()
