"""The paged library's boundary and refusals, without a GPU: everything here is turned away before a kernel is launched."""
import ctypes
import re
import subprocess
import zlib
from pathlib import Path

import pytest
import torch

import mistral_inference_b200 as mi
from mistral_inference_b200 import _abi_paged
from mistral_inference_b200.build import build_paged

from . import paged_util as U

REPO = Path(__file__).resolve().parents[1]
HEADER = REPO / "include" / "mistral_b200_paged.h"


@pytest.fixture(scope="module")
def lib():
    build_paged()
    return _abi_paged.lib()


def test_header_and_binding_name_the_same_symbols(lib):
    declared = set(re.findall(r"\b(mbp_[a-z0-9_]+)\s*\(", HEADER.read_text()))
    assert declared == set(_abi_paged._SIGNATURES)
    assert lib.mbp_abi_version() == _abi_paged.ABI_VERSION == int(re.search(r"MBP_ABI_VERSION (\d+)", HEADER.read_text()).group(1))


def test_constants_agree_with_the_header():
    text = HEADER.read_text()
    assert int(re.search(r"MBP_MAX_REQUESTS (\d+)", text).group(1)) == _abi_paged.MAX_REQUESTS
    assert f"top <= {_abi_paged.MAX_TOP}" in text


def last(lib):
    return lib.mbp_last_error().decode()


# Pointers that are never read: every call below is refused by its sizes.
X = 4096


def test_plans_are_refused(lib):
    extend = lambda B=2, T=2, R=2, P=4, N=8, rows=None, table=X: lib.mbp_pages_extend(table, X, X, X, X, rows, X, X, X, X, X, X, B, T, R, P, N, None)  # noqa: E731
    for kw, why in [(dict(table=None), "null"), (dict(B=0), "requests"), (dict(B=_abi_paged.MAX_REQUESTS + 1, R=5000), "requests"), (dict(B=3), "requests"), (dict(T=-1), "room"), (dict(T=2 ** 30 + 1), "room"), (dict(R=131073), "rows"),
                    (dict(R=0), "rows"), (dict(P=0), "pages"), (dict(N=0), "pages"), (dict(N=2 ** 31 // 64 + 1), "pages")]:
        assert extend(**kw) == -1 and why in last(lib), (kw, last(lib))
    truncate = lambda B=2, R=2, P=4, N=8, keep=X: lib.mbp_pages_truncate(X, X, X, X, X, None, keep, X, B, R, P, N, None)  # noqa: E731
    for kw, why in [(dict(keep=None), "null"), (dict(B=3), "requests"), (dict(R=0), "rows")]:
        assert truncate(**kw) == -1 and why in last(lib), (kw, last(lib))


def test_writes_are_refused(lib):
    def write(k=X, ldk=256, ldv=256, kv=X, B=1, T=1, KV=2, hd=128, N=4):
        return lib.mbp_pages_write(k, ldk, X, ldv, kv, X, X, X, X, B, T, KV, hd, N, None)
    for kw, why in [(dict(k=None), "null"), (dict(k=X + 8), "aligned"), (dict(ldk=128), "aligned"), (dict(ldv=260), "aligned"), (dict(kv=X + 4), "aligned"), (dict(hd=64), "128 only"),
                    (dict(B=0), "requests"), (dict(T=-1), "tokens"), (dict(KV=0), "heads"), (dict(N=2 ** 31 // 256), "heads")]:
        assert write(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert write(T=0) == 0


def test_attention_is_refused(lib):
    def attend(q=X, ldq=512, out=X, B=1, T=1, longest=1, most=0, H=4, KV=2, hd=128, P=4, N=4, window=0, scale=0.1, scratch=None, room=0):
        return lib.mbp_attn_pages(q, ldq, X, X, X, X, X, X, out, None, B, T, longest, most, 2, P, N, H, KV, hd, window, scale, scratch, room, None)
    for kw, why in [(dict(q=None), "null"), (dict(q=X + 4), "aligned"), (dict(ldq=256), "overlap"), (dict(H=5), "multiple"), (dict(H=66, ldq=66 * 128), "32 times"), (dict(hd=64), "128 only"),
                    (dict(out=X + 4), "aligned"), (dict(longest=0), "longest"), (dict(window=-1), "window"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(P=0), "P="), (dict(N=0), "pages")]:
        assert attend(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert attend(T=0) == 0
    scratch = lambda B=4, T=4000, longest=1000, most=0, P=64, H=32, KV=8, window=0: lib.mbp_attn_pages_scratch(B, T, longest, most, P, H, KV, window)  # noqa: E731
    need = scratch()  # (sized for 148 SMs where there is no GPU)
    assert need == 4 * 64 * 64 * 8 * 128 * 4 and scratch(longest=1) == 0 and scratch(T=40) == 0
    assert scratch(most=1500) < need and scratch(window=100) < need
    assert scratch(B=0) == scratch(T=0) == scratch(H=33) == scratch(KV=0) == scratch(window=-1) == 0
    assert 0 < scratch(B=64, T=64000, P=512) <= 1 << 30  # requests take turns
    for kw in (dict(scratch=None, room=need), dict(scratch=X, room=need - 1), dict(scratch=X + 16, room=need)):  # a portion without room
        assert attend(B=4, T=4000, longest=1000, P=64, H=32, KV=8, ldq=4096, **kw) == -2 and "scratch" in last(lib)


def test_scores_are_refused(lib):
    need = ctypes.c_int64(0)

    def score(logits=X, ld=100, dtype=1, target=X, logprob=X, T=2, V=100, top=3, scratch=X):
        return lib.mbp_token_scores(logits, ld, dtype, target, logprob, X, X, X, T, V, top, scratch, None)
    for kw, why in [(dict(logits=None), "null"), (dict(ld=99), "apart"), (dict(dtype=2), "dtype"), (dict(target=None), "null"), (dict(top=65), "top"), (dict(V=2, top=3), "top"), (dict(T=65536), "rows"),
                    (dict(scratch=X + 4), "null"), (dict(V=0), "vocab")]:
        assert score(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert score(T=0) == 0
    assert lib.mbp_token_scores_sizes(2, 100, 3, ctypes.byref(need)) == 0 and need.value > 0


def tables_cpu():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return i(2, 4), i(2), i(8), i(1)


def test_python_refuses_what_it_cannot_take():
    table, lens, free, n_free = tables_cpu()
    with pytest.raises(AssertionError):
        mi.PageTables(table.long(), lens, free, n_free)
    with pytest.raises(AssertionError):
        mi.PageTables(table, lens[:1], free, n_free)
    with pytest.raises(AssertionError):
        mi.PageTables(table[:, ::2], lens, free, n_free)
    with pytest.raises(AssertionError, match="CUDA"):  # no fallback
        mi.PageTables(table, lens, free, n_free)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    plan = mi.PagePlan(table, i(0), i(0, 1), i(0), i(0), i(0), 1)
    kv, scale = torch.zeros(4, 2, 2, 64, 128, dtype=torch.uint8), torch.ones(4, 2, 2)
    k, q = torch.zeros(1, 2, 128, dtype=torch.bfloat16), torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    for bad in (dict(kv=kv[:, :, :, :32]), dict(kv=kv.float()), dict(scale=scale.double()), dict(scale=scale[:, :1]), dict(k=k.float()), dict(k=k[:, :1]), dict(k=torch.cat([k, k]))):
        a = {**dict(kv=kv, scale=scale, k=k), **bad}
        with pytest.raises(AssertionError):
            mi.write_pages(a["kv"], a["scale"], a["k"], a["k"], plan)
    for bad in (dict(q=q[:, :3]), dict(q=q[0]), dict(q=q.half()), dict(out=torch.zeros(1, 512)), dict(q=torch.cat([q, q]))):
        a = {**dict(q=q, out=None), **bad}
        with pytest.raises(AssertionError):
            mi.attend_pages(a["q"], kv, scale, plan, out=a["out"])
    x = torch.zeros(2, 10)
    for bad in (dict(x=x.half()), dict(x=x[0]), dict(x=x.t()), dict(t=torch.zeros(2, dtype=torch.int32)), dict(t=torch.zeros(3, dtype=torch.long)), dict(top=11), dict(top=-1)):
        a = {**dict(x=x, t=None, top=1), **bad}
        with pytest.raises(AssertionError):
            mi.token_scores(a["x"], a["t"], top=a["top"])


def test_status_says_why():
    from mistral_inference_b200.paged import check_status
    check_status(torch.zeros(1, dtype=torch.int32))
    for code, word in ((1, "twice"), (2, "length"), (3, "room"), (4, "free"), (16, "wait"), (32, "most")):
        with pytest.raises(_abi_paged.Mb200Error, match=word):
            check_status(torch.tensor([code], dtype=torch.int32))


def test_the_restatement_rounds_like_torch():
    """The oracle's e4m3 against torch's own conversion, over every binade and the middles between codes."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(20000, generator=g) * torch.exp2(torch.randint(-12, 7, (20000,), generator=g).float())).clamp(-448, 448)
    grid = U.e4m3_grid().float()
    x = torch.cat([x, grid, -grid, (grid[1:] + grid[:-1]) / 2])
    assert torch.equal(U.to_e4m3(x.double()).float(), x.to(U.E4M3).float())


def test_host_tables_truncate_undoes_extend():
    t = U.HostTables(3, 8, 20)
    t.extend([100, 0, 65])
    before = (str(t.table), list(t.lens), list(t.free), t.n_free)
    t.extend([64, 1, 200])
    t.truncate([100, 0, 65])
    assert before == (str(t.table), t.lens, t.free, t.n_free)


def test_ledger_knows_what_there_is_room_for():
    from mistral_inference_b200.paged import PageLedger
    g = PageLedger(rows=3, max_seq_len=200, n_pages=5)
    g.admit(2)
    assert g.rows == [0, 1] and g.lens == [0, 0] and g.free_pages == 5
    g.check([130, 64])
    with pytest.raises(ValueError, match="4 of 5|more pages"):
        g.check([200, 130])
    for bad, why in (([1], "Batch size"), ([-1, 5], "new tokens"), ([0, 0], "new tokens"), ([201, 0], "200")):
        with pytest.raises(ValueError, match=why):
            g.check(bad)
    g.lens = [130, 64]
    assert g.free_pages == 1
    g.check([1, 1])  # one new page
    g.admit(1)
    with pytest.raises(ValueError, match="2 more pages needed, 1 of 5 free"):
        g.check([0, 1, 1])
    with pytest.raises(ValueError, match="free rows"):
        g.admit(1)
    g.retire([0])
    assert g.rows == [1, 2] and g.lens == [64, 0] and g.free_pages == 4
    g.admit(1)
    assert g.rows == [1, 2, 0]


def test_layered_decoders_keep_their_rings():
    from mistral_inference_b200.layered import LayeredTransformer
    with pytest.raises(ValueError, match="rings"):
        LayeredTransformer.make_cache(object(), 1, 8, kv_cache="pages")


def test_an_unknown_cache_is_refused():
    from mistral_inference_b200.transformer import Transformer
    for kw in (dict(kv_cache="paper"), dict(n_pages=3)):
        with pytest.raises(ValueError, match="kv_cache"):
            Transformer.make_cache(object(), 1, 8, **kw)


def test_declarations_of_this_abi_version():
    """A change of the declarations takes a new version, so that a library built before it is refused."""
    code = re.sub(r"/\*.*?\*/", " ", HEADER.read_text(), flags=re.S)
    assert zlib.crc32(" ".join(code.split()).encode()) == 1297119818, "raise the ABI version with this change"


def test_scratch_is_sized_by_the_device_that_the_call_runs_on(monkeypatch):
    """Devices of unlike size: what one of them needs is asked of it, and not taken from what another answered."""
    import contextlib
    current, asked = [0], []

    @contextlib.contextmanager
    def use(device):
        before, current[0] = current[0], device
        yield
        current[0] = before

    def sizes(*args):
        asked.append((current[0], args))
        return 1000 + current[0]

    monkeypatch.setattr(torch.cuda, "device", use)
    monkeypatch.setitem(_abi_paged._lazy, "mbp_attn_pages_scratch", sizes)
    _abi_paged._attn_scratch.cache_clear()
    try:
        sizes_of = [_abi_paged._attn_scratch(d, 2, 600, 300, 900, 20, 32, 8, 0) for d in (1, 0, 1)]
    finally:
        _abi_paged._attn_scratch.cache_clear()
    assert sizes_of == [1001, 1000, 1001] and [d for d, _ in asked] == [1, 0] and asked[0][1] == (2, 600, 300, 900, 20, 32, 8, 0)


def account(lens, on_device=None):
    """A PagedCache's account on the host, without its tensors."""
    from mistral_inference_b200.paged import PageLedger
    c = mi.PagedCache.__new__(mi.PagedCache)
    c.ledger = PageLedger(rows=4, max_seq_len=300, n_pages=20)
    c.ledger.admit(len(lens))
    c.ledger.lens, c._on_device, c.cache_sizes, c._started = list(lens), list(on_device or lens), [300, 300], True
    return c


def test_tokens_count_for_every_request_or_for_none():
    c = account([10, 20, 30], [11, 22, 30])
    for bad in ([1], [1, 2], [1, 2, 0, 0], [2, 0, 0], [-11, 0, 0]):
        with pytest.raises(AssertionError):
            c.update_seqlens(bad)
        assert c.ledger.lens == [10, 20, 30]
    c.update_seqlens([1, 1, -30])
    assert c.ledger.lens == [11, 21, 0]


def test_log_probabilities_of_requests_that_bring_nothing_are_refused():
    """Their last tokens' logits were those of memory that nobody wrote."""
    from types import SimpleNamespace
    from mistral_inference_b200.transformer import Transformer
    ids = torch.zeros(90, dtype=torch.long)
    for seqlens in ([0, 90], [90, 0], [40, 0, 50]):
        with pytest.raises(AssertionError, match="brings a token"):
            Transformer.forward_logprobs(SimpleNamespace(vocab_size=8, num_pipeline_ranks=1), ids, seqlens, account([5] * len(seqlens)), ids)


def test_numbers_of_alternatives_are_refused_before_the_prompt_runs():
    from types import SimpleNamespace

    def runs(*a, **kw):
        raise RuntimeError("the prompt ran")
    model = SimpleNamespace(device=torch.device("cpu"), args=SimpleNamespace(vocab_size=40, max_batch_size=1), make_cache=lambda *a, **kw: account([0]), forward_scores=runs, forward_logprobs=runs)
    model.eval = lambda: model
    for bad in (-1, 41, 65, 1000):
        with pytest.raises(ValueError, match="alternatives"):
            mi.generate([[1, 2]], model, max_tokens=1, temperature=0.0, alternatives=bad)
    for good in (0, 1, 40):
        with pytest.raises(RuntimeError, match="ran"):
            mi.generate([[1, 2]], model, max_tokens=1, temperature=0.0, alternatives=good)


LAYOUT = """
#include "plan_layout.cuh"
extern "C" void layout(int B, int R, int* out) {
  out[0] = mb200::plan_first_at(B); out[1] = mb200::plan_moved_at(B); out[2] = mb200::plan_named_at(B); out[3] = mb200::plan_named_words(R); out[4] = mb200::plan_words(B, R);
}
"""


def test_a_plans_shared_memory_holds_a_bit_for_every_row(tmp_path):
    """States have many more rows than a call has requests: one request of a server of thousands."""
    (tmp_path / "l.cc").write_text(LAYOUT)
    csrc = REPO / "mistral_inference_b200" / "csrc" / "paged"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", str(csrc), "-o", str(tmp_path / "l.so"), str(tmp_path / "l.cc")], check=True)
    layout, out = ctypes.CDLL(str(tmp_path / "l.so")).layout, (ctypes.c_int * 5)()
    for B in (1, 2, 3, 64, 1999, _abi_paged.MAX_REQUESTS):
        for R in (1, 2, 31, 32, 33, 128, 129, 300, 4000, 131071, 131072):
            layout(B, R, out)
            first, moved, named, named_words, words = out
            assert B <= first and first + B + 1 <= moved and moved + B + 1 <= words          # lengths, two prefix sums
            assert B <= named and 32 * named_words >= R and named + named_words <= words      # bits, which must not lie over the lengths
            assert 4 * words <= 48 * 1024 - 512                                               # beside the kernels' own few words
    text = (csrc / "paged_plan.cuh").read_text() + (csrc / "paged_abi.cu").read_text()
    assert "plan_words(p.B, p.R)" in text and text.count("plan_named_words(p.R)") == 1
