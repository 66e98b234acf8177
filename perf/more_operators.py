"""Performance cases of a tied head in microscaled 4-bit floating point
(MXFP4): quantisation, the rows of a table looked up again (embeddings), the
product with it, and the decode head with the sampling step behind it.

The format: a row's values in blocks of 32; a block has a scale 2^(s - 127), s
a byte (255: NaN), and 32 elements of 4 bits, two a byte, the first in the low
half: a sign, two bits of exponent and one of mantissa, 0 0.5 1 1.5 2 3 4 6.
Quantisation takes s - 127 = floor(log2(max |x|)) - 2, at least -127, and
rounds x / 2^(s - 127) to the nearest element, ties to the even one, past 6 to
6.  Codes lie row by row, 16 bytes a block, the scales beside them, a byte a
block, their rows padded to a multiple of four.

A case is a dict of plain values.  kind "quantize": [rows][dim] values quantised
and read back whole (what a program does that measures a table's error).
  x                f32 | bf16 | f16 values, y the type that they are read back in
kind "lookup": `rows` ids of a table [out][dim], read back
  y                f32 | bf16 | f16
kind "project": x [rows][dim] times a table [out][dim]
  x, y             f32 | bf16
  four             x is quantised first, its product one of 4-bit values
  softcap          cap * tanh(y / cap) behind the product (0: none)
kind "head": the logits of `rows` f32 hidden states [rows][dim], and a token of each
  temperature (0: greedy), top_k, top_p, softcap
"""
import math

import torch

own = False

QUANTIZE = {"kind": "quantize", "x": "bf16", "y": "bf16"}
LOOKUP = {"kind": "lookup", "y": "bf16"}
PROJECT = {"kind": "project", "x": "bf16", "y": "bf16", "four": False, "softcap": 0.0}
HEAD = {"kind": "head", "temperature": 1.0, "top_k": 50, "top_p": 0.9, "softcap": 0.0}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the hidden states of a chunk of prompts, before a product of 4-bit values
        dict(QUANTIZE, name="quantize_prompt", rows=2048, dim=4096),
        # a whole head laid out once, the largest vocabulary
        dict(QUANTIZE, name="quantize_table", rows=262144, dim=2560),
        # the embeddings of a batch's next tokens: latency
        dict(LOOKUP, name="lookup_batch", rows=128, dim=2560, out=262144),
        # the embeddings of a chunk of prompts, an odd vocabulary, f32 hidden states
        dict(LOOKUP, name="lookup_prompt", rows=8192, dim=2048, out=50257, y="f32"),
        # one request's token through an attention-sized projection: the smallest product, latency
        dict(PROJECT, name="token_projection", rows=1, dim=2560, out=2560),
        # the decode head of a small batch, the framework's f32 hidden states
        dict(PROJECT, name="head_small_batch", rows=16, dim=2560, out=151936, x="f32", y="f32"),
        # the decode head of a large batch over the largest vocabulary, capped logits
        dict(PROJECT, name="head_large_batch", rows=128, dim=2560, out=262144, y="f32", softcap=30.0),
        # a chunk of prompts against 4-bit weights
        dict(PROJECT, name="prompt_chunk", rows=2048, dim=4096, out=4096),
        # a batch's tokens, both sides of 4 bits, an odd number of rows and outputs
        dict(PROJECT, name="batch_four_bits", rows=61, dim=4096, out=11007, four=True),
        # chunks of prompts, both sides of 4 bits: the largest product
        dict(PROJECT, name="prompts_four_bits", rows=8192, dim=4096, out=11008, four=True),
        # the decode head of one chat over the largest vocabulary, sampled
        dict(HEAD, name="decode_head", rows=1, dim=2560, out=262144, softcap=30.0),
        # the rows of a speculative round, greedy
        dict(HEAD, name="verify_head", rows=3, dim=2560, out=248320, temperature=0.0, top_k=1, top_p=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "lookup", "project", "project", "project", "head"])
    if kind == "quantize":
        dim = _log(rng, 32, 16384)
        return dict(QUANTIZE, rows=max(1, min(_log(rng, 1, 262144), (262144 * 2560) // dim)), dim=dim,
                    x=rng.choice(["f32", "bf16", "bf16", "f16"]), y=rng.choice(["f32", "bf16"]))
    out = rng.choice([32000, 50257, 151936, 248320, 262144, _log(rng, 256, 262144), _log(rng, 256, 262144)])
    if kind == "lookup":
        dim = _log(rng, 32, 8192)
        return dict(LOOKUP, rows=_log(rng, 1, 16384), dim=dim, out=min(out, (262144 * 2560) // dim),
                    y=rng.choice(["f32", "bf16", "f16"]))
    if kind == "head":
        dim = 256 * rng.randint(2, 16)
        greedy = rng.random() < 0.3
        return dict(HEAD, rows=rng.randint(1, min(4, 12288 // dim)), dim=dim, out=min(out, (262144 * 2560) // dim),
                    temperature=0.0 if greedy else rng.choice([0.6, 1.0, 1.3]), top_k=rng.choice([1, 20, 50, 128]),
                    top_p=rng.choice([1.0, 0.9, 0.5]), softcap=rng.choice([0.0, 30.0]))
    four = rng.random() < 0.4
    dim = rng.choice([8, 32, 32]) * _log(rng, 8, 256)
    out, rows = min(out, (262144 * 2560) // dim), _log(rng, 1, 8192)
    rows = max(1, min(rows, int(6e11 / (dim * out)), (64 << 20) // out))
    return dict(PROJECT, rows=rows, dim=dim, out=out, four=four, x=rng.choice(["f32", "bf16", "bf16"]), y=rng.choice(["f32", "bf16"]),
                softcap=rng.choice([0.0, 0.0, 30.0]))


# ---------------------------------------------------------------- inputs --

class _State:
    pass


_tables = {}


def _table(name):
    """What a code, or a scale's byte, stands for."""
    if name not in _tables:
        half = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        values = half + [-v for v in half] if name == "code" else [2.0 ** (s - 127) for s in range(255)] + [math.nan]
        _tables[name] = torch.tensor(values, dtype=torch.float64).float().cuda()
    return _tables[name]


def _blocks(dim):
    return (dim + 31) // 32


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = _State()
    s.case = dict(case)
    rows, dim = case["rows"], case["dim"]
    if case["kind"] == "quantize":
        s.x = torch.empty((rows, dim), dtype=TYPES[case["x"]], device="cuda")
        s.x.normal_(0.0, 1.0, generator=g)
        s.x *= torch.exp(torch.randn((1, dim), generator=g, device="cuda")).to(s.x.dtype)  # columns differ, as channels do
        return s
    s.codes, s.scales = _weights(case["out"], dim, g)
    if case["kind"] == "lookup":
        s.ids = torch.randint(0, case["out"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        return s
    s.x = torch.randn((rows, dim), generator=g, device="cuda").to(TYPES[case.get("x", "f32")])  # final-normed: unit variance
    if case["kind"] == "head":
        s.uniforms = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    return s


def _weights(out, dim, g):
    """A table of normal values, as it lies in memory: codes and scales."""
    blocks = _blocks(dim)
    codes = torch.empty((out, 16 * blocks), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((out, (blocks + 3) // 4 * 4), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (32 * blocks))
    for at in range(0, out, step):
        n = min(step, out - at)
        w = torch.zeros((n, 32 * blocks), device="cuda")
        w[:, :dim].normal_(0.0, 2.0 / math.sqrt(dim), generator=g)
        codes[at:at + n], scales[at:at + n, :blocks] = _plain_codes(w.view(n, blocks, 32))
    return codes, scales


# ------------------------------------------------------------------ runs --

def run(state):
    return (_own if own else _plain)[state.case["kind"]](state)


_handle = None


def _sampler():
    global _handle
    if _handle is None:
        from shared_amd import Sampler
        _handle = Sampler(0)  # a program keeps one
    return _handle


def _held(s):
    from shared_amd import Mx4
    return Mx4(s.codes, s.scales, s.case["dim"])


def _own_quantize(s):
    h = _sampler()
    return h.lookup_mx4(h.quantize_mx4(s.x), out_dtype=TYPES[s.case["y"]])


def _own_lookup(s):
    return _sampler().lookup_mx4(_held(s), s.ids, out_dtype=TYPES[s.case["y"]])


def _own_project(s):
    h, c = _sampler(), s.case
    x = h.quantize_mx4(s.x) if c["four"] else s.x
    return h.project_mx4(x, _held(s), out_dtype=TYPES[c["y"]], softcap=c["softcap"])


def _own_head(s):
    from shared_amd import Params
    c = s.case
    r = _sampler().lm_head_sample(s.x, _held(s), logits=True, uniforms=s.uniforms,
                                  params=Params(temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], softcap=c["softcap"]))
    return {"ids": r["ids"], "logits": r["logits"]}


_own = {"quantize": _own_quantize, "lookup": _own_lookup, "project": _own_project, "head": _own_head}


def _plain_codes(x):
    """Codes [n][16 blocks] and scales [n][blocks] of x [n][blocks][32], f32."""
    top = x.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)
    t = x.abs() * _table("scale")[127 - e.clamp(max=126)]
    # the step between elements: 0.5 up to 2, 1 up to 4, then 2
    step = torch.where(t < 2, 0.5, torch.where(t < 4, 1.0, 2.0))
    q = (torch.round(t / step) * step).clamp(max=6.0)
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(x).to(torch.uint8)
    return (code[:, :, 0::2] + 16 * code[:, :, 1::2]).view(x.shape[0], -1), (e[:, :, 0] + 127).to(torch.uint8)


def _plain_values(codes, scales, dim):
    """f32 values [n][dim] of a table's rows."""
    n, blocks = codes.shape[0], _blocks(dim)
    pair = codes.view(n, blocks, 16).int()
    v = _table("code")[torch.stack((pair & 15, pair >> 4), 3)].view(n, blocks, 32)
    return (v * _table("scale")[scales[:, :blocks].int()][:, :, None]).view(n, 32 * blocks)[:, :dim]


def _plain_quantized(x):
    """x as f32 after quantisation."""
    n, dim = x.shape
    blocks = _blocks(dim)
    w = torch.zeros((n, 32 * blocks), device="cuda")
    w[:, :dim] = x
    codes, scales = _plain_codes(w.view(n, blocks, 32))
    return _plain_values(codes, scales, dim)


def _plain_quantize(s):
    return _plain_quantized(s.x).to(TYPES[s.case["y"]])


def _plain_lookup(s):
    ids = s.ids.long()
    return _plain_values(s.codes[ids], s.scales[ids], s.case["dim"]).to(TYPES[s.case["y"]])


def _plain_project(s):
    c = s.case
    x = _plain_quantized(s.x) if c["four"] else s.x.float()
    y = x @ _plain_values(s.codes, s.scales, c["dim"]).T
    if c["softcap"]:
        y = c["softcap"] * torch.tanh(y / c["softcap"])
    return y.to(TYPES[c["y"]])


def _plain_head(s):
    c = s.case
    logits = s.x @ _plain_values(s.codes, s.scales, c["dim"]).T
    v = c["softcap"] * torch.tanh(logits / c["softcap"]) if c["softcap"] else logits
    if c["temperature"] <= 0:
        return {"ids": v.argmax(1).to(torch.int32), "logits": logits}
    v, order = torch.sort(v, dim=1, descending=True, stable=True)
    k = min(c["top_k"], c["out"])
    p = torch.exp((v[:, :k].double() - v[:, :1].double()) / c["temperature"])
    mass = p.cumsum(1)
    # the fewest candidates whose share reaches top_p, then a draw among them in the order of their rank
    cut = ((mass / mass[:, -1:] < c["top_p"]).sum(1, keepdim=True) + 1).clamp(max=k)
    left = s.uniforms[:, None] * mass.gather(1, cut - 1)
    at = torch.minimum((mass < left).sum(1, keepdim=True), cut - 1)
    return {"ids": order.gather(1, at)[:, 0].to(torch.int32), "logits": logits}


_plain = {"quantize": _plain_quantize, "lookup": _plain_lookup, "project": _plain_project, "head": _plain_head}


def work(case):
    rows, dim = case["rows"], case["dim"]
    row4 = 17 * _blocks(dim)  # a quantised row
    if case["kind"] == "quantize":
        return {"bytes": rows * ((SIZE[case["x"]] + SIZE[case["y"]]) * dim + 2 * row4), "flops": 0}
    if case["kind"] == "lookup":
        return {"bytes": rows * (row4 + 4 + SIZE[case["y"]] * dim), "flops": 0}
    out = case["out"]
    if case["kind"] == "head":
        return {"bytes": out * row4 + rows * (4 * dim + 4 * out + 12), "flops": 2 * rows * dim * out}
    return {"bytes": out * row4 + rows * (SIZE[case["x"]] * dim + (2 * row4 if case["four"] else 0) + SIZE[case["y"]] * out),
            "flops": 2 * rows * dim * out}


# ------------------------------------------------- the definitions, 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"quantize": _exact_quantize, "lookup": _exact_lookup, "project": _exact_project, "head": _exact_head}[case["kind"]](s)


def _exact_rounded(x):
    """x [n][dim] as quantisation leaves it, by the borders between elements."""
    n, dim = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -dim % 32)).view(n, -1, 32)
    size = x.abs()
    top = size.max(2, keepdim=True).values
    unit = 2.0 ** torch.where(top > 0, (torch.log2(top) + 0.0).floor() - 2, -127.0).clamp(min=-127.0)
    size /= unit
    # borders, and whether a value on one goes up (to the even element)
    grid = torch.zeros_like(size)
    for border, up, element in ((0.25, False, 0.5), (0.75, True, 1.0), (1.25, False, 1.5), (1.75, True, 2.0), (2.5, False, 3.0),
                                (3.5, True, 4.0), (5.0, False, 6.0)):
        grid[(size >= border) if up else (size > border)] = element
    return (torch.copysign(grid, x) * unit).view(n, -1)[:, :dim]


def _exact_quantize(s):
    step = max(1, (1 << 25) // s.x.shape[1])
    return torch.cat([_exact_rounded(s.x[at:at + step]) for at in range(0, s.x.shape[0], step)])


def _exact_rows(codes, scales, dim):
    pair = torch.stack((codes % 16, codes // 16), 2).view(codes.shape[0], -1)[:, :dim].double()
    low, e = pair % 2, (pair % 8 // 2)
    size = torch.where(e > 0, (1 + low / 2) * 2.0 ** (e - 1), low / 2)
    unit = torch.repeat_interleave(2.0 ** (scales[:, :_blocks(dim)].double() - 127), 32, dim=1)[:, :dim]
    return torch.where(pair >= 8, -size, size) * unit


def _exact_lookup(s):
    ids = s.ids.long()
    return _exact_rows(s.codes[ids], s.scales[ids], s.case["dim"])


def _exact_product(s, x):
    out, dim = s.case["out"], s.case["dim"]
    y = torch.empty((x.shape[0], out), dtype=torch.float64, device="cuda")
    for at in range(0, out, 16384):
        y[:, at:at + 16384] = x @ _exact_rows(s.codes[at:at + 16384], s.scales[at:at + 16384], dim).T
    return y


def _exact_project(s):
    cap = s.case["softcap"]
    y = _exact_product(s, _exact_rounded(s.x) if s.case["four"] else s.x.double())
    return torch.tanh(y / cap) * cap if cap else y


def _exact_head(s):
    c = s.case
    logits = _exact_product(s, s.x.double())
    v = torch.tanh(logits / c["softcap"]) * c["softcap"] if c["softcap"] else logits
    ids = []
    for r in range(v.shape[0]):
        k = min(c["top_k"], c["out"]) if c["temperature"] > 0 else 1
        top, at = (t.cpu() for t in torch.topk(v[r], k))
        if c["temperature"] <= 0:
            ids.append(int(at[0]))
            continue
        p = [math.exp((float(x) - float(top[0])) / c["temperature"]) for x in top]
        total, run_, cut = sum(p), 0.0, k
        for i in range(k):
            run_ += p[i] / total
            if run_ >= c["top_p"]:
                cut = i + 1
                break
        left, i = float(s.uniforms[r]) * sum(p[:cut]), 0
        while i < cut - 1 and left - p[i] > 0:
            left -= p[i]
            i += 1
        ids.append(int(at[i]))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "logits": logits}
