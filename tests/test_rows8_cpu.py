"""The boundary and refusals of libmb200_rows8, without a GPU: everything here is turned away before a kernel is launched."""
import re
import types
from pathlib import Path

import pytest
import torch

import mistral_inference_b200 as mi
from mistral_inference_b200 import _abi_rows8
from mistral_inference_b200 import _abi, rows8 as operators
from mistral_inference_b200.build import build_rows8
from mistral_inference_b200.rows8 import Rows8

from . import rows8_util as U

REPO = Path(__file__).resolve().parents[1]
HEADER = REPO / "include" / "mistral_b200_rows8.h"


@pytest.fixture(scope="module")
def lib():
    build_rows8()
    return _abi_rows8.lib()


def test_header_and_binding_name_the_same_symbols(lib):
    declared = set(re.findall(r"\b(mb8_[a-z0-9_]+)\s*\(", HEADER.read_text()))
    assert declared == set(_abi_rows8._SIGNATURES)
    assert lib.mb8_abi_version() == _abi_rows8.ABI_VERSION == int(re.search(r"MB8_ABI_VERSION (\d+)", HEADER.read_text()).group(1))


def test_constants_agree_with_the_header():
    text = HEADER.read_text()
    assert int(re.search(r"MB8_MAX_NORM (\d+)", text).group(1)) == _abi_rows8.MAX_NORM
    assert 1 << int(re.search(r"MB8_MAX_ROWS \(1 << (\d+)\)", text).group(1)) == _abi_rows8.MAX_ROWS


def last(lib):
    return lib.mb8_last_error().decode()


# Pointers that are never read: every call below is refused by its sizes.
X = 4096
BIG = (1 << 24) + 1


def test_quantise_is_refused(lib):
    def call(x=X, ld=256, dtype=0, codes=X, scales=X, T=2, K=256):
        return lib.mb8_quantise(x, ld, dtype, codes, scales, T, K, None)
    for kw, why in [(dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=X + 8), "16 bytes"), (dict(scales=X + 4), "16 bytes"), (dict(x=X + 1), "aligned"),
                    (dict(x=X + 2, dtype=1), "aligned"), (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(ld=255), "apart"), (dict(T=-1), "rows"), (dict(K=0), "entries"),
                    (dict(T=BIG), "rows"), (dict(K=BIG, ld=BIG), "entries")]:
        assert call(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert call(T=0, x=None) == 0


def test_norm_is_refused(lib):
    def call(x=X, ld=256, add=X, ld_add=256, w=X, dtype=0, out=X, codes=X, scales=X, T=2, K=256):
        return lib.mb8_norm(x, ld, add, ld_add, w, dtype, out, codes, scales, T, K, 1e-5, None)
    for kw, why in [(dict(x=None), "null"), (dict(w=None), "null"), (dict(out=None), "null"), (dict(codes=None), "null"), (dict(ld=255), "apart"), (dict(ld_add=255), "apart"),
                    (dict(add=X + 1), "aligned"), (dict(w=X + 1), "aligned"), (dict(dtype=2), "dtype"), (dict(K=65537, ld=65537, ld_add=65537), "65536"), (dict(T=-1), "rows"), (dict(K=0), "entries")]:
        assert call(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert call(T=0, x=None) == 0


def test_products_are_refused(lib):
    def multiply(xc=X, xs=X, wc=X, ws=X, out=X, ld=64, dtype=0, T=2, N=64, K=256):
        return lib.mb8_multiply(xc, xs, wc, ws, out, ld, dtype, T, N, K, 0, None, 0, None)
    for kw, why in [(dict(xc=None), "null"), (dict(xs=None), "null"), (dict(wc=None), "null"), (dict(ws=None), "null"), (dict(out=None), "null"), (dict(xc=X + 8), "16 bytes"), (dict(ws=X + 1), "16 bytes"),
                    (dict(out=X + 1), "aligned"), (dict(out=X + 2, dtype=1), "aligned"), (dict(dtype=2), "dtype"), (dict(ld=63), "apart"), (dict(T=-1), "rows"), (dict(N=0), "features"), (dict(K=0), "entries"),
                    (dict(T=BIG), "rows"), (dict(N=BIG, ld=BIG), "features"), (dict(K=BIG), "entries")]:
        assert multiply(**kw) == -1 and why in last(lib), (kw, last(lib))

    def gate(xc=X, xs=X, wc=X, ws=X, codes=X, scales=X, T=2, H=64, K=256):
        return lib.mb8_gate(xc, xs, wc, ws, codes, scales, T, H, K, 0, None, 0, None)
    for kw, why in [(dict(xc=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=X + 8), "16 bytes"), (dict(T=-1), "rows"), (dict(H=0), "features"),
                    (dict(H=(1 << 23) + 1), "features"), (dict(K=0), "entries")]:
        assert gate(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert multiply(T=0, out=None, xc=None) == gate(T=0, codes=None, xc=None) == 0


def test_sizes_whose_doubles_are_no_sizes_are_refused(lib):
    for H in (-(2 ** 63) + 1, -(2 ** 63) + 64, 2 ** 62 + 1, 2 ** 63 - 1):
        assert lib.mb8_gate(X, X, X, X, X, X, 2, H, 256, 0, None, 0, None) == -1 and "features" in last(lib), H
    for heads, kv in ((1, 2 ** 62 + 5), (1, 2 ** 63 - 1), (2 ** 63 - 1, 1), (2 ** 63 - 4, 2 ** 62)):
        assert lib.mb8_rotate(X, X, X, None, X, X, X, 2, heads, kv, None) == -1 and "heads" in last(lib), (heads, kv)
    for sizes in ((2 ** 62, 256, 256), (300, 2 ** 62, 256), (300, 256, 2 ** 62), (300, 2 ** 63 - 1, 2 ** 63 - 1)):
        assert lib.mb8_product_scratch(*sizes) == 0


def test_rotate_is_refused(lib):
    def call(qkv=X, rope=X, positions=X, q=X, k=X, v=X, T=2, heads=4, kv=2):
        return lib.mb8_rotate(qkv, rope, positions, None, q, k, v, T, heads, kv, None)
    for kw, why in [(dict(qkv=None), "null"), (dict(rope=None), "null"), (dict(positions=None), "null"), (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(q=X + 8), "16 bytes"),
                    (dict(T=-1), "tokens"), (dict(T=BIG), "tokens"), (dict(heads=0), "heads"), (dict(kv=0), "heads"), (dict(heads=65535), "heads")]:
        assert call(**kw) == -1 and why in last(lib), (kw, last(lib))
    assert call(T=0, qkv=None) == 0


def rows(R, K):
    return Rows8.empty(R, K, "cpu")


def test_python_refuses_what_does_not_fit():
    bf = dict(dtype=torch.bfloat16)
    for x in [torch.zeros(3, 4, dtype=torch.float16), torch.zeros(4, **bf), torch.zeros(2, 0, **bf), torch.zeros(4, 6, **bf).t(), torch.zeros(1, 6, **bf).expand(3, 6), torch.zeros(4, 6, **bf)]:
        with pytest.raises(AssertionError):  # (the last one for its device)
            mi.quantise_rows(x)
    with pytest.raises(AssertionError):
        mi.multiply_rows(rows(2, 100), rows(3, 100))
    with pytest.raises(AssertionError):
        Rows8.empty(2, 0, "cpu")
    with pytest.raises(AssertionError):
        Rows8.empty(2, BIG, "cpu")


@pytest.mark.parametrize("dtype,other", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_results_of_another_type_than_asked_for_are_refused(dtype, other):
    with pytest.raises(AssertionError, match="of another"):
        mi.multiply_rows(rows(2, 9), rows(3, 9), dtype=dtype, out=torch.zeros(2, 3, dtype=other))
    for said in (None, dtype):
        with pytest.raises(AssertionError, match="no fallback"):
            mi.multiply_rows(rows(2, 9), rows(3, 9), dtype=said, out=torch.zeros(2, 3, dtype=dtype))


def test_what_is_no_tensor_is_refused():
    bf = torch.zeros(2, 3, dtype=torch.bfloat16)
    for call in (lambda: mi.quantise_rows(None), lambda: mi.quantise_rows([[1.0]]), lambda: mi.norm_rows(bf, None, 1e-5), lambda: mi.multiply_rows(Rows8(None, None, 3), rows(3, 9)),
                 lambda: mi.gate_rows(rows(2, 9), Rows8(rows(4, 9).codes, 7, 9))):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: mi.multiply_rows(rows(2, 9), Rows8(rows(3, 9).codes, rows(3, 9).scales, "9")), lambda: mi.multiply_rows(None, rows(3, 9))):
        with pytest.raises((AssertionError, TypeError, AttributeError)):
            call()


def test_no_cpu_fallback():
    for call in (lambda: mi.quantise_rows(torch.zeros(2, 3)), lambda: mi.norm_rows(torch.zeros(2, 3), torch.zeros(3), 1e-5), lambda: mi.multiply_rows(rows(2, 9), rows(3, 9)),
                 lambda: mi.gate_rows(rows(2, 9), rows(4, 9))):
        with pytest.raises(AssertionError, match="no fallback"):
            call()


@pytest.mark.parametrize("R,K", [(1, 1), (130, 1003), (128, 512), (33, 4096), (300, 640)])
def test_numbers_and_exponents(R, K):
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(R)) * torch.exp2(torch.randint(-20, 20, (R, K), generator=torch.Generator().manual_seed(K)).float())
    codes, scales = U.quantised(x)
    r = Rows8(codes, scales.view(torch.float8_e8m0fnu), K)
    assert torch.equal(r.numbers(torch.float64), U.numbers(codes, scales, K)) and torch.equal(r.exponents().long(), U.exponent(U.blocks_of(x).abs().amax(2)))
    empty = Rows8.empty(R, K, "cpu")
    assert empty.codes.shape == codes.shape and empty.scales.shape == scales.shape and empty.rows == R
    # half a step, 2^-4 of a number, or 2^-10 of the power among the smallest
    size = U.power(U.exponent(U.blocks_of(x).abs().amax(2))).repeat_interleave(128, 1)[:, :K]
    assert ((r.numbers(torch.float64) - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, size * 2.0 ** -10)).all()


@pytest.mark.parametrize("K", [1, 300])
def test_numbers_and_exponents_of_no_rows(K):
    r = rows(0, K)
    assert r.numbers().shape == r.numbers(torch.bfloat16).shape == (0, K) and r.exponents().shape == (0, -(-K // 128))


def test_the_restatement_refuses_wrong_rows():
    """What the GPU tests hold results to, held to mistakes: a code, a power, a place of no row."""
    x = torch.randn(40, 300, generator=torch.Generator().manual_seed(1)).double()
    codes, scales = U.quantised(x.float())
    U.assert_rows_near(codes, scales, x.float().double(), 0.0)
    wrong = codes.clone().view(torch.uint8)
    wrong[7, 200] ^= 8
    with pytest.raises(AssertionError):
        U.assert_rows_near(wrong.view(torch.float8_e4m3fn), scales, x.float().double(), 0.0)
    for at in [(0, 0, 3, 0, 1), (0, 0, 20, 1, 0), (0, 0, 0, 0, 3)]:
        wrong = scales.clone()
        wrong[at] += 1
        with pytest.raises(AssertionError):
            U.assert_rows_near(codes, wrong, x.float().double(), 0.0)


def test_powers_of_any_byte():
    """Scales that another program wrote: 2^-127, the largest, and the byte that is no number."""
    r = rows(4, 128)
    r.codes.copy_(torch.full((4, 128), 1.5).to(torch.float8_e4m3fn))
    bytes_ = r.scales.view(torch.uint8)
    bytes_.fill_(127)
    for i, b in enumerate((0, 1, 254, 255)):
        bytes_[0, 0, i, 0, 0] = b
    x = r.numbers(torch.float64)
    assert (x[0] == 1.5 * 2.0 ** -127).all() and (x[1] == 1.5 * 2.0 ** -126).all() and (x[2] == 1.5 * 2.0 ** 127).all() and x[3].isnan().all()
    assert r.exponents().tolist() == [[-127], [-126], [127], [128]]


def test_command_line_refuses_8_bits_of_other_designs(tmp_path):
    from mistral_inference_b200.main import main
    (tmp_path / "config.json").write_text('{"architecture": "Fesenex"}')
    with pytest.raises(SystemExit):
        main(["generate", str(tmp_path), "--prompt", "1", "--weights", "e4m3"])


# ----------------------------------------------------------------------------------------------------- a model's weights
class Failing:
    """quantise_rows of a GPU that has memory for `room` matrices; rows that nobody reads."""

    def __init__(self, room):
        self.room = room

    def __call__(self, x):
        if self.room == 0:
            raise torch.OutOfMemoryError("no room")
        self.room -= 1
        return rows(x.shape[0], x.shape[1])


@pytest.fixture
def model(monkeypatch):
    """A model on the CPU that takes itself to be on a GPU: what is tested here ends before anything is launched there."""
    from mistral_inference_b200.transformer import Transformer
    args = mi.TransformerArgs(dim=64, n_layers=3, head_dim=16, hidden_dim=96, n_heads=4, n_kv_heads=2, norm_eps=1e-5, vocab_size=80, max_batch_size=2)
    m = Transformer.empty(args, "cpu", torch.bfloat16)
    monkeypatch.setattr(Transformer, "device", property(lambda self: torch.device("cuda")))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    return m


def refusals(m):
    cache = types.SimpleNamespace(paged=False, _kv_seqlens_host=[5], cache_sizes=[9])
    one = torch.zeros(1, dtype=torch.long)
    return [lambda: m.forward(one, [1]), lambda: m.forward(one, [1], cache), lambda: m.forward_partial(one, [1]), lambda: m.decode_static(one, cache), lambda: m.next_token_logits(one, cache),
            lambda: m.forward_logprobs(one, [1], None, one), lambda: m.forward_scores(one, [1], None, one, 2), m.state_dict, lambda: m.load_state_dict({}),
            lambda: m._load_lora_state_dict({"lora": torch.zeros(1, dtype=torch.bfloat16)})]


@pytest.mark.parametrize("room", [4, 7, 12])  # at the second layer's first matrix, its last one, and the head
def test_weights_that_were_quantised_half_way(model, monkeypatch, room):
    """Memory that ends on the way leaves matrices of both kinds: nothing runs on them, until a second call has gone on behind the first."""
    monkeypatch.setattr(operators, "quantise_rows", Failing(room))
    with pytest.raises(torch.OutOfMemoryError):
        model.quantise_weights(head=True)
    done = [layer.attention.wqkv8 for layer in model.layers.values()]
    assert [d is not None for d in done] == [room >= 4, room >= 8, room >= 12] and not model.weights8
    for call in refusals(model):
        with pytest.raises(_abi.Mb200Error, match="8 bits"):
            call()
    monkeypatch.setattr(operators, "quantise_rows", Failing(13))
    assert model.quantise_weights(head=True) is model and model.weights8
    for layer, before in zip(model.layers.values(), done):
        assert before is None or layer.attention.wqkv8 is before
        for r, n, k in ((layer.attention.wqkv8, 128, 64), (layer.attention.wo8, 64, 64), (layer.feed_forward.w13_8, 192, 64), (layer.feed_forward.w2_8, 64, 96)):
            assert r.fixed and (r.rows, r.cols) == (n, k)
    assert model._output8.fixed and model.output_weight.numel() == 0
    with pytest.raises(_abi.Mb200Error, match="already"):
        model.quantise_weights()
    with pytest.raises(_abi.Mb200Error, match="8 bits"):
        model.state_dict()


def test_weights_of_which_none_was_quantised(model, monkeypatch):
    """Memory that ends at the first layer has changed nothing."""
    monkeypatch.setattr(operators, "quantise_rows", Failing(3))
    with pytest.raises(torch.OutOfMemoryError):
        model.quantise_weights()
    model._check_runnable()
    assert len(model.state_dict()) == 3 + 3 * 9 and all(v.numel() > 0 for v in model.state_dict().values())


def test_8_bit_matrices_follow_a_model(model, monkeypatch):
    """To another device with the parameters; a conversion of these leaves codes and scales as they are."""
    monkeypatch.setattr(operators, "quantise_rows", Failing(100))
    model.quantise_weights(head=True)
    monkeypatch.undo()

    def kept():
        return [model._output8] + [r for b in model.layers.values() for r in (b.attention.wqkv8, b.attention.wo8, b.feed_forward.w13_8, b.feed_forward.w2_8)]
    before = kept()
    model.to("cpu").float().bfloat16()
    assert all(a is b for a, b in zip(before, kept()))
    model.to("meta")
    for a, b in zip(before, kept()):
        assert b.codes.device.type == b.scales.device.type == "meta" and (b.rows, b.cols) == (a.rows, a.cols) and (b.codes.dtype, b.scales.dtype) == (a.codes.dtype, a.scales.dtype)
        assert not b.fixed


def test_steps_captured_before_a_move_are_not_replayed():
    from mistral_inference_b200.transformer import Transformer
    args = mi.TransformerArgs(dim=64, n_layers=1, head_dim=16, hidden_dim=96, n_heads=4, n_kv_heads=2, norm_eps=1e-5, vocab_size=80)
    m, cache = Transformer.empty(args, "cpu", torch.bfloat16), types.SimpleNamespace()
    first = m._decode_state(cache, "step")
    assert m.to("cpu")._decode_state(cache, "step") is first  # (nothing moved)
    m.float().bfloat16()
    assert m._decode_state(cache, "step") is not first


def test_a_move_that_fails_on_its_way_is_gone_on_with(model, monkeypatch):
    """Matrices that are left behind move with the next call, and nothing captured before the first one is replayed behind it."""
    monkeypatch.setattr(operators, "quantise_rows", Failing(100))
    model.quantise_weights()
    monkeypatch.undo()
    own, room = Rows8.to, [5]

    def to(self, device):
        room[0] -= 1
        if room[0] < 0:
            raise torch.OutOfMemoryError("no room")
        return own(self, device)
    monkeypatch.setattr(Rows8, "to", to)
    moves = model._moves
    with pytest.raises(torch.OutOfMemoryError):
        model.to("meta")
    assert model._moves > moves
    monkeypatch.undo()
    devices = [getattr(owner, name).codes.device.type for owner, name in model._matrices8()]
    assert devices == ["meta"] * 5 + ["cpu"] * 7
    model.to("meta")
    assert {getattr(owner, name).codes.device.type for owner, name in model._matrices8()} == {"meta"}
