"""The grouped and the microscaled 4-bit products as they are measured: cases, inputs, plain forms.

Layouts are those of the library's C ABI: matrices are column-major, so a torch tensor of shape (rows, K),
contiguous, is the K x rows column-major matrix.  The kinds of cases:

* ``grouped``    out[t] = W[g(t)] x[t], tokens sorted by group (ragged columns; forward and, with the weights read
                 the other way round, input gradient)
* ``grouped_k``  grad[e] = alpha * sum over the tokens t of group e of outer(dy[t], x[t]) + beta * C[e]
* ``quantize``   blocks of 32 values -> 4-bit elements and a shared power of two, and back to values
* ``mx``         product of two 4-bit operands
* ``mx_grouped`` ``grouped`` with 4-bit weights and tokens; ``fresh`` quantises the tokens inside the call

Plain forms are elementary torch operations in 32 bits; a group's rows are padded to the longest group so that all
groups are one batched product.
"""
import functools
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one step of serving: eight tokens, each at an expert of its own; the experts' weights are what is read
        dict(name="grouped decode", kind="grouped", tokens=8, groups=64, M=1024, K=2048, trans=True, ab="bf16", out="bf16", skew=0.0, tail=0),
        # a training or prefill batch, routed unevenly
        dict(name="grouped forward", kind="grouped", tokens=16384, groups=32, M=2048, K=4096, trans=True, ab="bf16", out="bf16", skew=0.7, tail=0),
        # the gradient of the tokens of such a batch, an odd number of them, with unused rows behind the last group
        dict(name="grouped input grad", kind="grouped", tokens=10007, groups=16, M=2048, K=1408, trans=False, ab="f16", out="f32", skew=0.7, tail=121),
        # the gradient of the weights, added to what earlier batches left
        dict(name="grouped weight grad", kind="grouped_k", tokens=16384, groups=32, M=2048, N=1408, ab="bf16", out="f32", beta=1.0, skew=0.7),
        # the same for a short batch: many experts, some of them without a token
        dict(name="grouped weight grad short", kind="grouped_k", tokens=1501, groups=64, M=512, N=768, ab="bf16", out="bf16", beta=0.0, skew=1.0),
        # activations of one layer on their way into a 4-bit product
        dict(name="quantize activations", kind="quantize", rows=333, K=4096, x="bf16", trans=False),
        # a weight matrix stored the other way round, with a ragged last block
        dict(name="quantize weights", kind="quantize", rows=8192, K=8190, x="f16", trans=True),
        # one token through one 4-bit layer
        dict(name="mx token", kind="mx", M=8192, N=1, K=8192, out="bf16", beta=0.0),
        # the benchmark's square product in 4 bits
        dict(name="mx square", kind="mx", M=8192, N=8192, K=8192, out="bf16", beta=0.0),
        # sizes that fill no tile, a Float32 result added to another
        dict(name="mx ragged", kind="mx", M=4100, N=1111, K=4128, out="f32", beta=1.0),
        # one step of serving a mixture of 4-bit experts
        dict(name="mx grouped decode", kind="mx_grouped", tokens=48, groups=32, M=2048, K=4096, out="bf16", skew=0.5, fresh=False),
        # its prefill, from 16-bit tokens
        dict(name="mx grouped prefill", kind="mx_grouped", tokens=16384, groups=32, M=4096, K=2048, out="bf16", skew=0.7, fresh=True),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["grouped", "grouped", "grouped_k", "quantize", "mx", "mx_grouped", "mx_grouped"])
    skew = rng.choice([0.0, 0.3, 0.7, 1.0])
    if kind == "grouped":
        return dict(kind=kind, tokens=_log(rng, 1, 16384), groups=_log(rng, 1, 64), M=_log(rng, 64, 4096, 8), K=_log(rng, 64, 4096, 8),
                    trans=rng.random() < 0.6, ab=rng.choice(["bf16", "f16"]), out=rng.choice(["bf16", "f16", "f32"]), skew=skew,
                    tail=rng.choice([0, 0, 1, 77]))
    if kind == "grouped_k":
        return dict(kind=kind, tokens=_log(rng, 1, 16384), groups=_log(rng, 1, 64), M=_log(rng, 64, 2048, 8), N=_log(rng, 64, 2048, 8),
                    ab=rng.choice(["bf16", "f16"]), out=rng.choice(["bf16", "f32", "f32"]), beta=rng.choice([0.0, 1.0]), skew=skew)
    if kind == "quantize":
        return dict(kind=kind, rows=_log(rng, 1, 8192), K=_log(rng, 32, 8192), x=rng.choice(["bf16", "f16", "f32"]), trans=rng.random() < 0.4)
    if kind == "mx":
        return dict(kind=kind, M=_log(rng, 64, 8192, 4), N=_log(rng, 1, 8192), K=_log(rng, 32, 8192, 32), out=rng.choice(["bf16", "f16", "f32"]),
                    beta=rng.choice([0.0, 0.0, 1.0]))
    return dict(kind=kind, tokens=_log(rng, 1, 16384), groups=_log(rng, 1, 32), M=_log(rng, 64, 4096, 8), K=_log(rng, 64, 4096, 32),
                out=rng.choice(["bf16", "f16", "f32"]), skew=skew, fresh=rng.random() < 0.5)


def work(case):
    c = case
    if c["kind"] == "quantize":
        n = c["rows"] * c["K"]
        # values in; elements and scales out and in again; values out
        return {"bytes": n * (BYTES[c["x"]] + 2 * 17 / 32 + BYTES[c["x"]]), "flops": 4 * n}
    if c["kind"] == "mx":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": 17 / 32 * K * (M + N) + M * N * (BYTES[c["out"]] + (4 if c["beta"] else 0)), "flops": 2 * M * N * K}
    T, E, M = c["tokens"], c["groups"], c["M"]
    if c["kind"] == "grouped_k":
        N = c["N"]
        return {"bytes": 2 * T * (M + N) + E * M * N * (BYTES[c["out"]] + (4 if c["beta"] else 0)), "flops": 2 * T * M * N}
    used = E * (1 - (1 - 1 / E) ** T)  # groups that get a token, were the routing even
    if c["kind"] == "grouped":
        return {"bytes": 2 * used * M * c["K"] + T * (2 * c["K"] + M * BYTES[c["out"]]), "flops": 2 * T * M * c["K"]}
    return {"bytes": 17 / 32 * used * M * c["K"] + T * (c["K"] * (2 if c["fresh"] else 17 / 32) + M * BYTES[c["out"]]), "flops": 2 * T * M * c["K"]}


# ------------------------------------------------------------------------------------------------------------------
# the 4-bit format
# ------------------------------------------------------------------------------------------------------------------
# Elements: sign, 2 exponent bits, 1 fraction bit.  A block of 32 along K shares 2^(s - 127), s an 8-bit code (255 is NaN).
# Two elements a byte, the first in the low half.  Scales lie in tiles of 128 rows x 4 blocks: row r and block b of a tile at
# byte (r % 32) * 16 + (r // 32) * 4 + b; tiles go along K first.  Groups of rows begin with a tile of their own.
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _up(n, m):
    return (n + m - 1) // m * m


def _power(e):
    """2^e in 32 bits for whole e from -127 to 127, from its bit pattern: a power function may be a bit off."""
    return torch.where(e == -127, 1 << 22, (e.int() + 127) << 23).int().view(torch.float32)


def _quantized(x):
    """(element codes, scale codes) of the rows of x, K a multiple of 32: blocks of 32, nearest element, ties to even."""
    v = x.float().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    e = torch.clamp(torch.frexp(top).exponent - 3, -127, 127)
    e = torch.where(top == 0, torch.full_like(e, -127), e)
    u = v * _power(-e)
    a = u.abs()
    near = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.clamp(torch.round(a / 2), max=3) + 4))
    codes = near.to(torch.uint8) | (torch.signbit(u).to(torch.uint8) << 3)
    return codes.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _values(codes, scales):
    """float32 values of element codes (rows, K) and scale codes (rows, K / 32)."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float32, device=codes.device)
    power = torch.where(scales == 255, torch.full((), float("nan"), device=codes.device), _power(torch.clamp(scales.int() - 127, max=127)))
    return (grid[codes.long()].unflatten(-1, (-1, 32)) * power.unsqueeze(-1)).flatten(-2)


def _packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpacked(bytes_):
    return torch.stack((bytes_ & 15, bytes_ >> 4), -1).flatten(-2)


def _tiled(scales):
    """(..., rows, blocks) with rows a multiple of 128 -> tiles; blocks are filled up to whole tiles with 0."""
    pad = _up(scales.shape[-1], 4) - scales.shape[-1]
    s = torch.nn.functional.pad(scales, (0, pad))
    s = s.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))  # tile row, r // 32, r % 32, tile column, block
    return s.movedim(-2, -4).transpose(-3, -2).contiguous()  # tile row, tile column, r % 32, r // 32, block


def _untiled(tiles, blocks):
    """Back to (..., rows, blocks)."""
    s = tiles.transpose(-3, -2).movedim(-4, -2)  # tile row, r // 32, r % 32, tile column, block
    return s.flatten(-5, -3).flatten(-2)[..., :blocks]


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _sizes(case, seed):
    """Tokens per group: an uneven routing drawn from the seed."""
    r = np.random.RandomState(seed % (1 << 32))
    p = np.exp(case["skew"] * r.standard_normal(case["groups"]))
    return r.multinomial(case["tokens"], p / p.sum())


def _offsets(n):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).to(DEVICE)


def _place(off, T):
    """Group of each token and its place in the group, and whether it belongs to one."""
    t = torch.arange(T, device=off.device)
    g = torch.searchsorted(off[1:].contiguous(), t.int(), right=True)
    inside = g < off.numel() - 1
    g = torch.clamp(g, max=off.numel() - 2)
    return g, torch.where(inside, t - off[g], 0), inside


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda shape, scale=1.0: torch.randn(shape, generator=gen, device=DEVICE) * scale  # noqa: E731
    kind = c["kind"]
    s = {"case": c}
    if kind == "quantize":
        R, K = c["rows"], c["K"]
        # channels differ in size, as those of activations and weights do
        x = normal((R, K)) * torch.exp(normal((1, K)))
        x = x.to(TYPES[c["x"]])
        s["x"] = x.t().contiguous() if c["trans"] else x
        s["q"] = torch.empty((R, _up(K, 32) // 2), dtype=torch.uint8, device=DEVICE)
        s["s"] = torch.empty((_up(R, 128) // 128 * _up(K, 128) // 128 * 512,), dtype=torch.uint8, device=DEVICE)
        s["y"] = torch.empty((R, K), dtype=TYPES[c["x"]], device=DEVICE)
        return s
    if kind == "mx":
        M, N, K = c["M"], c["N"], c["K"]
        s["a"], s["sa"] = _operand(normal((M, K), K ** -0.5))
        s["b"], s["sb"] = _operand(normal((N, K)))
        s["c"] = normal((N, M)) if c["beta"] else None
        s["d"] = torch.empty((N, M), dtype=TYPES[c["out"]], device=DEVICE)
        return s
    n = _sizes(c, seed)
    T, E, M = c["tokens"], c["groups"], c["M"]
    s["offsets"], s["longest"] = _offsets(n), int(n.max())
    if kind == "grouped_k":
        N = c["N"]
        s["x"] = normal((T, N)).to(TYPES[c["ab"]])
        s["dy"] = normal((T, M), 0.02).to(TYPES[c["ab"]])
        s["c"] = normal((E, N, M)) if c["beta"] else None
        s["d"] = torch.empty((E, N, M), dtype=TYPES[c["out"]], device=DEVICE)
        return s
    K = c["K"]
    if kind == "grouped":
        w = normal((E, M, K), K ** -0.5).to(TYPES[c["ab"]])
        s["w"] = w if c["trans"] else w.transpose(1, 2).contiguous()
        s["x"] = normal((T + c["tail"], K)).to(TYPES[c["ab"]])
        s["d"] = normal((T + c["tail"], M)).to(TYPES[c["out"]])  # what lies behind the last group stays
        return s
    w, sw = zip(*[_operand(normal((M, K), K ** -0.5)) for _ in range(E)])
    s["w"], s["sw"] = torch.stack(w), torch.stack(sw)
    x = normal((T, K)).to(torch.bfloat16)
    codes, scales = _quantized(x)
    g, place, _ = _place(s["offsets"], T)
    tiles = (s["offsets"][1:] - s["offsets"][:-1] + 127) // 128
    first = torch.cumsum(tiles, 0) - tiles
    s["rows"] = first[g] * 128 + place  # of each token's scales
    full = torch.zeros(((T + 127 * E) // 128 * 128, K // 32), dtype=torch.uint8, device=DEVICE)
    full[s["rows"]] = scales
    s["x"], s["q"], s["sq"] = x, _packed(codes), _tiled(full)
    s["d"] = torch.empty((T, M), dtype=TYPES[c["out"]], device=DEVICE)
    return s


def _operand(x):
    """Packed elements and tiled scales of one matrix (rows, K)."""
    codes, scales = _quantized(x)
    full = torch.zeros((_up(x.shape[0], 128), scales.shape[1]), dtype=torch.uint8, device=x.device)
    full[: x.shape[0]] = scales
    return _packed(codes), _tiled(full)


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _by_group(x, off, longest):
    """Rows of x as (groups, longest, width), zero behind a group's last row."""
    at = torch.arange(longest, device=x.device)
    start, n = off[:-1].long().unsqueeze(1), (off[1:] - off[:-1]).unsqueeze(1)
    rows = torch.clamp(start + at, max=x.shape[0] - 1)
    return torch.where((at < n).unsqueeze(-1), x[rows], 0)


def _grouped(x, w, s, out):
    """out[t] = w[g(t)] x[t] for the tokens of a group; the other rows of out stay."""
    y = torch.bmm(_by_group(x, s["offsets"], s["longest"]), w.transpose(1, 2))
    g, place, inside = _place(s["offsets"], out.shape[0])
    return torch.where(inside.unsqueeze(1), y[g, place].to(out.dtype), out)


def _plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        x = s["x"].t() if c["trans"] else s["x"]
        K = c["K"]
        codes, scales = _quantized(torch.nn.functional.pad(x, (0, _up(K, 32) - K)))
        return _values(codes, scales)[:, :K].to(s["y"].dtype)
    if kind == "mx":
        a = _values(_unpacked(s["a"]), _untiled(s["sa"], c["K"] // 32)[: c["M"]])
        b = _values(_unpacked(s["b"]), _untiled(s["sb"], c["K"] // 32)[: c["N"]])
        d = b @ a.t()
        return (d if s["c"] is None else d + c["beta"] * s["c"]).to(s["d"].dtype)
    if kind == "grouped_k":
        x, dy = (_by_group(s[k].float(), s["offsets"], s["longest"]) for k in ("x", "dy"))
        d = torch.bmm(x.transpose(1, 2), dy)
        return (d if s["c"] is None else d + c["beta"] * s["c"]).to(s["d"].dtype)
    if kind == "grouped":
        w = s["w"].float()
        return _grouped(s["x"].float(), w if c["trans"] else w.transpose(1, 2), s, s["d"])
    if c["fresh"]:
        x = _values(*_quantized(s["x"]))
    else:
        x = _values(_unpacked(s["q"]), _untiled(s["sq"], c["K"] // 32)[s["rows"]])
    w = _values(_unpacked(s["w"]).flatten(0, 1), _untiled(s["sw"], c["K"] // 32)[:, : c["M"]].flatten(0, 1))
    return _grouped(x, w.unflatten(0, (c["groups"], c["M"])), s, s["d"])


@functools.lru_cache(maxsize=None)
def _library(device):
    import __graft_entry__

    __graft_entry__.load_package()
    from cudanative_jl_b200.bfloat16 import BFloat16
    from cudanative_jl_b200.gemm import Handle

    return Handle(device), {torch.bfloat16: BFloat16, torch.float16: np.float16, torch.float32: np.float32}


def _own(s):
    c = s["case"]
    kind = c["kind"]
    h, tag = _library(torch.cuda.current_device())
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda k: s[k].data_ptr()  # noqa: E731
    if kind == "quantize":
        R, K, x = c["rows"], c["K"], s["x"]
        t, ldq = tag[x.dtype], _up(K, 32)
        h.mxfp4_quantize(c["trans"], K, R, at("x"), x.stride(0), t, at("q"), ldq, at("s"), stream=stream)
        h.mxfp4_dequantize(K, R, at("q"), ldq, at("s"), at("y"), K, t, stream=stream)
        return s["y"]
    if kind == "mx":
        M, N, K = c["M"], c["N"], c["K"]
        h.gemm_mxfp4(M, N, K, 1.0, at("a"), K, at("sa"), at("b"), K, at("sb"), c["beta"], at("c") if c["beta"] else None, M,
                     np.float32, at("d"), M, tag[s["d"].dtype], stream=stream)
        return s["d"]
    E, M, off = c["groups"], c["M"], at("offsets")
    if kind == "grouped_k":
        N = c["N"]
        h.gemm_grouped_k(M, N, c["tokens"], 1.0, at("dy"), M, at("x"), N, tag[s["x"].dtype], c["beta"], at("c") if c["beta"] else None, M,
                         M * N, np.float32, at("d"), M, M * N, tag[s["d"].dtype], off, E, stream=stream)
        return s["d"]
    K, out = c["K"], tag[s["d"].dtype]
    if kind == "grouped":
        h.gemm_grouped(c["trans"], M, c["tokens"] + c["tail"], K, 1.0, at("w"), K if c["trans"] else M, M * K, at("x"), K, tag[s["x"].dtype],
                       0.0, None, M, out, at("d"), M, out, off, E, stream=stream)
        return s["d"]
    T = c["tokens"]
    if c["fresh"]:
        h.mxfp4_quantize(False, K, T, at("x"), K, tag[s["x"].dtype], at("q"), K, at("sq"), offsets=off, groups=E, stream=stream)
    h.gemm_mxfp4_grouped(M, T, K, 1.0, at("w"), K, M * K, at("sw"), at("q"), K, at("sq"), 0.0, None, M, out, at("d"), M, out, off, E,
                         stream=stream)
    return s["d"]


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def _powers64(device):
    return torch.tensor([math.ldexp(1.0, e) for e in range(-127, 128)], dtype=torch.float64, device=device)


def _nearest64(x):
    """The values, in 64 bits, that the 4-bit blocks of the rows of x stand for."""
    K = x.shape[1]
    v = torch.zeros((x.shape[0], _up(K, 32)), dtype=torch.float64, device=x.device)
    v[:, :K] = x.double()
    v = v.view(x.shape[0], -1, 32)
    top = v.abs().max(-1, keepdim=True).values
    powers = _powers64(x.device)  # the largest that is not above the block's top, and two steps down
    power = powers[torch.clamp(torch.searchsorted(powers, top, right=True) - 3, 0, 254)]
    a = v.abs() / power
    step = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    return (torch.sign(v) * grid[step] * power).view(x.shape[0], -1)[:, :K]


def _decoded64(packed, tiles, row):
    """The values of packed elements (rows, K / 2) whose scales lie at tile rows `row`, from the bit fields."""
    b = packed.long()
    codes = torch.empty((b.shape[0], 2 * b.shape[1]), dtype=torch.int64, device=b.device)
    codes[:, 0::2], codes[:, 1::2] = b % 16, b // 16
    exponent, fraction = codes // 2 % 4, codes % 2
    size = torch.where(exponent == 0, 0.5 * fraction, (1 << torch.clamp(exponent - 1, min=0)) * (1 + 0.5 * fraction))
    v = torch.where(codes >= 8, -size, size).double()
    block = torch.arange(v.shape[1], device=b.device) // 32
    flat, per_row = tiles.reshape(-1), tiles.shape[-4]
    where = ((row // 128).unsqueeze(1) * per_row + block // 4) * 512 + (row % 32 * 16 + row % 128 // 32 * 4).unsqueeze(1) + block % 4
    return v * _powers64(b.device)[flat[where].long()]


def exact(case, seed):
    s, c = prepare(case, seed), case
    kind = c["kind"]
    if kind == "quantize":
        return _nearest64(s["x"].t() if c["trans"] else s["x"])
    if kind == "mx":
        a = _decoded64(s["a"], s["sa"], torch.arange(c["M"], device=DEVICE))
        b = _decoded64(s["b"], s["sb"], torch.arange(c["N"], device=DEVICE))
        return b @ a.t() + (c["beta"] * s["c"].double() if c["beta"] else 0)
    edges = s["offsets"].tolist()
    spans = list(zip(edges[:-1], edges[1:]))
    if kind == "grouped_k":
        d = torch.stack([s["x"][i:j].double().t() @ s["dy"][i:j].double() for i, j in spans])
        return d + (c["beta"] * s["c"].double() if c["beta"] else 0)
    out = s["d"].double()
    if kind == "mx_grouped":
        x = _nearest64(s["x"]) if c["fresh"] else _decoded64(s["q"], s["sq"], s["rows"].long())
    for e, (i, j) in enumerate(spans):
        if kind == "grouped":
            w = s["w"][e].double()
            out[i:j] = s["x"][i:j].double() @ (w.t() if c["trans"] else w)
        else:
            out[i:j] = x[i:j] @ _decoded64(s["w"][e], s["sw"][e], torch.arange(c["M"], device=DEVICE)).t()
    return out
