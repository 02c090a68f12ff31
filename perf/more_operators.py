"""Operators of a transformer whose Linears multiply 8-bit numbers, as cases that can be timed and checked:

  quantise  rows of numbers to e4m3 codes with a scale (a power of two) for every 128 entries of a row
  norm      root-mean-square norm of a residual stream, with the addition to the stream ahead of it, its output in that form
  multiply  the product of two matrices in that form, tokens [T, K] by weights [N, K], to 16 or 32 bits
  gate      the product with interleaved gate and up weights [2 H, K], silu(gate) * up behind it, its output in that form again

Codes are [rows, K rounded up to 128] of e4m3, zeros behind a row's K entries.  Scales are 8-bit exponents (e8m0) in tiles of 128 rows by 4 blocks of 128 entries, as the
tensor cores read them: [row tiles, block tiles, 32, 4, 4], row 32 j + i and block b of a tile at [i, j, b]; places of no row or no block hold 1.  Shapes are those
of this repository's configurations and generic ones."""
import math
import types
import zlib

import torch

own = False

DEV = "cuda"
BLOCK = 128
E4M3_MAX = 448.0
LOWEST_EXP = -100  # exponent of the scale of a block of zeros

# width, width of the feed-forward's hidden layer, rows of the query, key and value weights, vocabulary
SHAPES = {"7b": (4096, 14336, 6144, 32000), "nemo": (5120, 14336, 6144, 131072), "8x22b": (6144, 16384, 8192, 32768), "odd": (1003, 2777, 1555, 5003)}


def listed():
    return [
        # attention's results of a decode step of 32 requests, ahead of the output weights
        {"name": "quantise_b32", "kind": "quantise", "T": 32, "K": 4096, "dtype": "bf16"},
        # gate and up weights of a layer, while a checkpoint is loaded
        {"name": "quantise_weights", "kind": "quantise", "T": 28672, "K": 4096, "dtype": "bf16"},
        # chat with one user: the norm between a sublayer and the next
        {"name": "norm_7b_b1", "kind": "norm", "T": 1, "K": 4096, "add": 1, "dtype": "bf16"},
        # 8 prompts of 1000 tokens
        {"name": "norm_nemo_t8000", "kind": "norm", "T": 8000, "K": 5120, "add": 1, "dtype": "bf16"},
        # chat with one user: query, key and value weights
        {"name": "multiply_7b_b1", "kind": "multiply", "T": 1, "K": 4096, "N": 6144, "out": "bf16"},
        # a decode step of 32 requests: the feed-forward's way down
        {"name": "multiply_nemo_b32", "kind": "multiply", "T": 32, "K": 14336, "N": 5120, "out": "bf16"},
        # a step's logits of eight requests
        {"name": "multiply_head_b8", "kind": "multiply", "T": 8, "K": 4096, "N": 32000, "out": "fp32"},
        # a portion of a prompt: query, key and value weights
        {"name": "multiply_7b_t777", "kind": "multiply", "T": 777, "K": 4096, "N": 6144, "out": "bf16"},
        # a prompt of 4096 tokens: the feed-forward's way down
        {"name": "multiply_7b_t4096", "kind": "multiply", "T": 4096, "K": 14336, "N": 4096, "out": "bf16"},
        # chat with one user: into the feed-forward
        {"name": "gate_7b_b1", "kind": "gate", "T": 1, "K": 4096, "H": 14336},
        # drafted tokens of eight requests, six each
        {"name": "gate_nemo_b48", "kind": "gate", "T": 48, "K": 5120, "H": 14336},
        # a prompt of 4096 tokens
        {"name": "gate_7b_t4096", "kind": "gate", "T": 4096, "K": 4096, "H": 14336},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Widths of this repository's configurations under half of the time, any others the rest."""
    kind = rng.choice(["quantise", "norm", "multiply", "multiply", "multiply", "gate", "gate"])
    known = rng.random() < 0.4
    width, hidden, qkv, vocab = SHAPES[rng.choice(sorted(SHAPES))]
    few = rng.random() < 0.6
    tokens = _log(rng, 3 if known else 1, 64) if few else _log(rng, 65, 4000)
    if kind == "quantise":
        return {"kind": kind, "T": _log(rng, 1, 16000), "K": rng.choice([width, hidden]) if known else _log(rng, 1, 6000), "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    if kind == "norm":
        return {"kind": kind, "T": _log(rng, 2, 8000), "K": width if known else _log(rng, 16, 9000), "add": rng.choice([0, 1, 1]), "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    if kind == "multiply":
        K, N, out = rng.choice([(width, qkv, "bf16"), (width, width, "bf16"), (hidden, width, "bf16"), (width, vocab, "fp32")]) if known else (_log(rng, 16, 9000), _log(rng, 64, 16000), rng.choice(["bf16", "fp32"]))
        return {"kind": kind, "T": min(tokens, 64) if N > 16000 else tokens, "K": K, "N": N, "out": out}
    K, H = (width, hidden) if known else (_log(rng, 16, 9000), _log(rng, 64, 12000))
    return {"kind": kind, "T": min(tokens, 4096 * 14336 * 4096 // (K * H)), "K": K, "H": H}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed, name):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003) ^ zlib.crc32(name.encode()))


def _normal(seed, name, shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=_generator(seed, name))


def _spread(seed, name, n):
    """Sizes of n channels: most alike, a few of them many times as large."""
    g = _generator(seed, name)
    size = torch.exp2(torch.randint(-1, 2, (n,), device=DEV, generator=g).float())
    return torch.where(torch.rand(n, device=DEV, generator=g) < 0.003, size * 24, size)


def prepare(case, seed):
    st = types.SimpleNamespace(case=case, kind=case["kind"], eps=1e-5)
    T, K = case["T"], case["K"]
    x = _normal(seed, "x", (T, K), 0.9) * _spread(seed, "channels", K)
    if st.kind in ("quantise", "norm"):
        dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        st.x = x.to(dtype)
        if st.kind == "norm":
            st.weight = (1 + _normal(seed, "weight", (K,), 0.1)).to(dtype)
            st.add = _normal(seed, "add", (T, K), 0.3).to(dtype) if case["add"] else None
        return st
    rows = case["N"] if st.kind == "multiply" else 2 * case["H"]
    st.x_codes, st.x_scales = _plain_quantise(x)
    st.w_codes, st.w_scales = _plain_quantise(_normal(seed, "w", (rows, K), 1.4 * K ** -0.5))  # (quantised when the checkpoint is loaded)
    st.out = torch.float32 if case.get("out") == "fp32" else torch.bfloat16
    return st


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _up(n, step):
    return -(-n // step) * step


def _exponent(amax):
    """The exponent of a block's scale: the smallest e with amax <= 448 * 2^e, at least LOWEST_EXP (as whole numbers)."""
    mantissa, e = torch.frexp(amax)  # amax = mantissa * 2^e, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(amax > 0, e - 9 + (mantissa > 0.875).int(), LOWEST_EXP).clamp(min=LOWEST_EXP)


def _power(e):
    """2^e exactly, of whole numbers e that 32-bit numbers have."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _blocks(x):
    """[T, K] as [T, blocks, 128], zeros behind the end."""
    T, K = x.shape
    out = x.new_zeros(T, _up(K, BLOCK))
    out[:, :K] = x
    return out.view(T, -1, BLOCK)


def _tiled(e):
    """Exponents [T, blocks] as tiles of 8-bit ones."""
    T, n = e.shape
    out = torch.zeros(_up(T, 128), _up(n, 4), dtype=torch.int32, device=e.device)
    out[:T, :n] = e
    out = (out + 127).to(torch.uint8).view(-1, 4, 32, _up(n, 4) // 4, 4)
    return out.permute(0, 3, 2, 1, 4).contiguous().view(torch.float8_e8m0fnu)


def _untiled(scales, T, n):
    """Exponents [T, n] out of tiles."""
    tiles, quads = scales.shape[:2]
    return scales.view(torch.uint8).permute(0, 3, 2, 1, 4).reshape(tiles * 128, quads * 4)[:T, :n].int() - 127


def _plain_quantise(x):
    b = _blocks(x.float())
    e = _exponent(b.abs().amax(2))
    return (b * _power(-e)[:, :, None]).to(torch.float8_e4m3fn).view(x.shape[0], -1), _tiled(e)


def _plain_values(codes, scales):
    T, width = codes.shape
    e = _untiled(scales, T, width // BLOCK)
    return (codes.float().view(T, -1, BLOCK) * _power(e)[:, :, None]).view(T, width)


def _plain_norm(st):
    h = st.x.float()
    if st.add is not None:
        h = (h + st.add.float()).to(st.x.dtype)
    y = h.float() * torch.rsqrt(h.float().square().mean(1, keepdim=True) + st.eps) * st.weight.float()
    codes, scales = _plain_quantise(y)
    return {"codes": codes, "scales": scales, "stream": h.to(st.x.dtype)}


def _plain_product(st):
    return torch.matmul(_plain_values(st.x_codes, st.x_scales), _plain_values(st.w_codes, st.w_scales).t())


def _plain(st):
    if st.kind == "quantise":
        codes, scales = _plain_quantise(st.x)
        return {"codes": codes, "scales": scales}
    if st.kind == "norm":
        return _plain_norm(st)
    y = _plain_product(st)
    if st.kind == "multiply":
        return y.to(st.out)
    gate, up = y[:, 0::2], y[:, 1::2]
    codes, scales = _plain_quantise(gate / (1 + torch.exp(-gate)) * up)
    return {"codes": codes, "scales": scales}


# ------------------------------------------------------------------------------------------------------------------ the framework's calls
def _own(st):
    from mistral_inference_b200.rows8 import Rows8, gate_rows, multiply_rows, norm_rows, quantise_rows
    if st.kind == "quantise":
        r = quantise_rows(st.x)
        return {"codes": r.codes, "scales": r.scales}
    if st.kind == "norm":
        r, stream = norm_rows(st.x, st.weight, st.eps, add=st.add)
        return {"codes": r.codes, "scales": r.scales, "stream": stream}
    K = st.case["K"]
    x, w = Rows8(st.x_codes, st.x_scales, K), Rows8(st.w_codes, st.w_scales, K)
    if st.kind == "multiply":
        return multiply_rows(x, w, dtype=st.out)
    r = gate_rows(x, w)
    return {"codes": r.codes, "scales": r.scales}


def run(st):
    return _own(st) if own else _plain(st)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    T, K = case["T"], case["K"]
    if case["kind"] == "quantise":
        return {"bytes": T * K * ((4 if case["dtype"] == "fp32" else 2) + 1 + 1 / BLOCK), "flops": 3 * T * K}  # magnitude, maximum, product
    if case["kind"] == "norm":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * K * (size * (1 + 2 * case["add"]) + 1 + 1 / BLOCK) + size * K, "flops": (7 + case["add"]) * T * K}
    rows = case["N"] if case["kind"] == "multiply" else 2 * case["H"]
    out = T * rows * (4 if case["out"] == "fp32" else 2) if case["kind"] == "multiply" else T * case["H"] * (1 + 1 / BLOCK)
    return {"bytes": (T + rows) * K * (1 + 1 / BLOCK) + out, "flops": 2 * T * rows * K}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_scale(y):
    """2^e [T, blocks] of rows in 64 bits, e found by comparisons with powers of two."""
    T, K = y.shape
    amax = torch.nn.functional.pad(y, (0, -K % BLOCK)).view(T, -1, BLOCK).abs().amax(2) / E4M3_MAX
    powers = torch.tensor([2.0 ** e for e in range(LOWEST_EXP, 128)], dtype=torch.float64, device=y.device)
    return powers[torch.searchsorted(powers, amax.contiguous()).clamp(max=len(powers) - 1)]


def _exact_rows(y):
    """What the codes stand for before their rounding, and the scales in their places."""
    T, K = y.shape
    size = _exact_scale(y)
    codes = torch.nn.functional.pad(y, (0, -K % BLOCK)) / size.repeat_interleave(BLOCK, 1)
    n = size.shape[1]
    r, b = torch.meshgrid(torch.arange(T, device=y.device), torch.arange(n, device=y.device), indexing="ij")
    tiles = torch.ones(-(-T // 128), -(-n // 4), 32, 4, 4, dtype=torch.float64, device=y.device)
    tiles[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = size
    return {"codes": codes, "scales": tiles}


def _exact_values(codes, scales, T, K):
    wide = scales.double()  # [tiles, quads, 32, 4, 4]
    r, b = torch.meshgrid(torch.arange(T, device=codes.device), torch.arange(-(-K // BLOCK), device=codes.device), indexing="ij")
    size = wide[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]
    return codes[:, :K].double() * size.repeat_interleave(BLOCK, 1)[:, :K]


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "quantise":
        return _exact_rows(st.x.double())
    if case["kind"] == "norm":
        h = st.x.double()
        if st.add is not None:
            h = (h + st.add.double()).to(st.x.dtype).double()  # (the stream is kept in its type)
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + st.eps) * st.weight.double()
        return {**_exact_rows(y), "stream": h}
    T, K = case["T"], case["K"]
    rows = case["N"] if case["kind"] == "multiply" else 2 * case["H"]
    y = _exact_values(st.x_codes, st.x_scales, T, K) @ _exact_values(st.w_codes, st.w_scales, rows, K).t()
    if case["kind"] == "multiply":
        return y
    return _exact_rows(y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2])
