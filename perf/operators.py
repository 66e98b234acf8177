"""Performance cases of the multi-adapter decode head: a shared projection
with the low-rank adapters of many requests beside it, and sampling with
temperature, top-k, top-p and min-p over the whole vocabulary.

A case is a dict of plain values.  kind "project":
  rows, dim, out   x [rows][dim] times the shared weight [out][dim], bf16
  adapters, rank   the pool: a [adapters][rank][dim], b [adapters][out][rank], bf16
  ragged           every adapter uses a rank of its own, 1 .. rank
  plain_share      share of the rows that use no adapter
  grouped          rows of a request are neighbours (prompts), else shuffled
  x, y             types of the hidden states and of the result: f32 | bf16
  softcap          cap * tanh(y / cap) behind the projection (0: none)
kind "sample":
  rows, vocab, logits   f32 | bf16 | f16 logits [rows][vocab]
  temperature, top_k (0: off), top_p (1: off), min_p (0: off)
  repetition, presence, frequency, history   penalties over each row's ids
  mixed            every row has parameters of its own around these
  density          allowed share of a grammar's mask (0: no mask)
  spread           peaked (few likely ids over a noisy floor, as a language
                   model gives) | flat (a wide normal, as at high entropy)

The plain forms compute in 32 bits, but for the masses exp((v - max) / T) and
their sums: token ids are whole numbers that have to come out the same, and
sums of 262,144 masses in 32 bits move a draw by more than the rarest ids
weigh.  (The plain sampling's time is its sort's.)
"""
import math

import numpy as np
import torch

own = False

PROJECT = {"kind": "project", "ragged": False, "plain_share": 0.0, "grouped": False, "x": "bf16", "y": "f32", "softcap": 0.0}
SAMPLE = {"kind": "sample", "logits": "f32", "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "repetition": 1.0,
          "presence": 0.0, "frequency": 0.0, "history": 0, "mixed": False, "density": 0.0, "spread": "peaked"}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PARAMS = np.dtype([("temperature", "<f8"), ("top_p", "<f8"), ("min_p", "<f8"), ("repetition_penalty", "<f8"),
                   ("presence_penalty", "<f8"), ("frequency_penalty", "<f8"), ("softcap", "<f4"), ("top_k", "<i4")])


def listed():
    return [
        # one request's token through an attention-sized projection: the smallest call, latency
        dict(PROJECT, name="token_projection", rows=1, dim=2560, out=2560, adapters=8, rank=16, y="bf16"),
        # the decode head of a small batch, the framework's f32 hidden states
        dict(PROJECT, name="head_small_batch", rows=16, dim=2560, out=151936, adapters=4, rank=16, x="f32"),
        # the decode head of a large batch over the largest vocabulary, capped logits
        dict(PROJECT, name="head_large_batch", rows=128, dim=2560, out=262144, adapters=16, rank=16, softcap=30.0,
             plain_share=0.25),
        # as many adapters as requests, ranks of their own, an odd number of rows and outputs
        dict(PROJECT, name="adapter_each", rows=61, dim=4096, out=11007, adapters=61, rank=64, ragged=True, y="bf16"),
        # a chunk of prompts, rows of a request together: matrix products
        dict(PROJECT, name="prompt_chunk", rows=2048, dim=4096, out=4096, adapters=6, rank=32, grouped=True, y="bf16"),
        # hidden states in f32, more rows than one tile, an odd vocabulary
        dict(PROJECT, name="head_f32_rows", rows=200, dim=2048, out=50257, adapters=32, rank=8, x="f32"),
        # one chat: latency
        dict(SAMPLE, name="one_row", rows=1, vocab=151936, temperature=0.7, top_p=0.9, min_p=0.05),
        # an ordinary batch with min-p alone, bf16 logits
        dict(SAMPLE, name="batch_min_p", rows=64, vocab=151936, logits="bf16", min_p=0.08),
        # a large batch under a grammar, nucleus over the whole vocabulary
        dict(SAMPLE, name="batch_top_p_grammar", rows=128, vocab=262144, top_p=0.95, density=0.3),
        # the largest batch, nothing cut off (sampling for training data)
        dict(SAMPLE, name="batch_unfiltered", rows=256, vocab=262144),
        # requests with parameters and histories of their own, an odd vocabulary
        dict(SAMPLE, name="mixed_requests", rows=37, vocab=50257, temperature=0.9, top_k=200, top_p=0.95, min_p=0.02,
             repetition=1.1, presence=0.5, frequency=0.2, history=300, mixed=True),
        # high entropy: thousands of ids are kept
        dict(SAMPLE, name="flat_wide_nucleus", rows=32, vocab=128256, logits="f16", temperature=1.3, top_k=20000, top_p=0.98,
             spread="flat"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        dim, out, rows = 8 * _log(rng, 32, 1024), _log(rng, 256, 262144), _log(rng, 1, 4096)
        out = min(out, (128 << 18) * 2560 // dim // 128)
        rows = max(1, min(rows, int(64e9 / (dim * out)), (64 << 20) // out))
        n = rng.choice([1, 4, _log(rng, 1, 64), min(rows, 64)])
        return dict(PROJECT, rows=rows, dim=dim, out=out, adapters=n, rank=rng.choice([8, 16, 16, 32, 64]),
                    ragged=rng.random() < 0.3, plain_share=rng.choice([0.0, 0.0, 0.25, 0.9]), grouped=rng.random() < 0.3,
                    x=rng.choice(["f32", "bf16", "bf16"]), y=rng.choice(["f32", "bf16"]), softcap=rng.choice([0.0, 0.0, 30.0]))
    vocab = rng.choice([32000, 50257, 128256, 151936, 248320, 262144, _log(rng, 1000, 262144), _log(rng, 1000, 262144)])
    return dict(SAMPLE, rows=min(_log(rng, 1, 256), max(1, (200 << 18) // vocab)), vocab=vocab,
                logits=rng.choice(["f32", "f32", "bf16", "f16"]), temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.4]),
                top_k=rng.choice([0, 0, 50, _log(rng, 1, vocab)]), top_p=rng.choice([1.0, 0.9, 0.95, rng.uniform(0.3, 0.999)]),
                min_p=rng.choice([0.0, 0.05, rng.uniform(0.001, 0.3)]), repetition=rng.choice([1.0, 1.1]),
                presence=rng.choice([0.0, 0.5]), frequency=rng.choice([0.0, 0.2]), history=rng.choice([0, 0, _log(rng, 8, 4096)]),
                mixed=rng.random() < 0.3, density=rng.choice([0.0, 0.0, 0.05, 0.5]),
                spread=rng.choice(["peaked", "peaked", "flat"]))


# ---------------------------------------------------------------- inputs --

class _State:
    pass


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = _State()
    s.case = dict(case)
    (_prepare_project if case["kind"] == "project" else _prepare_sample)(s, case, g, rng)
    return s


def _users(case):
    """Rows that use an adapter, and how many adapters they use."""
    rows = case["rows"] - int(case["rows"] * case["plain_share"])
    return rows, min(rows, case["adapters"])


def _prepare_project(s, case, g, rng):
    rows, dim, out, n, rank = (case[k] for k in ("rows", "dim", "out", "adapters", "rank"))

    def normal(shape, sigma):
        t = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        t.normal_(0.0, sigma, generator=g)
        return t

    s.x = torch.randn((rows, dim), generator=g, device="cuda").to(TYPES[case["x"]])  # final-normed: unit variance
    s.weight = normal((out, dim), 2.0 / math.sqrt(dim))
    s.a = normal((n, rank, dim), 1.0 / math.sqrt(dim))
    s.b = normal((n, out, rank), 0.5 / math.sqrt(rank))
    s.scales = torch.from_numpy(rng.uniform(0.5, 2.0, n).astype(np.float32)).cuda()
    s.ranks = torch.from_numpy((rng.integers(1, rank + 1, n) if case["ragged"] else np.full(n, rank)).astype(np.int32)).cuda()
    users, _ = _users(case)
    which = np.full(rows, -1, dtype=np.int32)
    which[:users] = np.arange(users) % n
    which = np.sort(which) if case["grouped"] else rng.permutation(which)
    s.row_adapter = torch.from_numpy(which.astype(np.int32)).cuda()


def _prepare_sample(s, case, g, rng):
    rows, vocab = case["rows"], case["vocab"]
    if case["spread"] == "flat":
        v = torch.randn((rows, vocab), generator=g, device="cuda") * 3.0
    else:
        # a floor of unlikely ids, and likely ones whose mass falls as a power of their rank
        v = torch.randn((rows, vocab), generator=g, device="cuda") * 1.8
        hot = max(1, min(2000, vocab // 4))
        rank = torch.arange(1, hot + 1, device="cuda", dtype=torch.float32)
        steep = 1.0 + torch.rand((rows, 1), generator=g, device="cuda")
        top = 16.0 + 6.0 * torch.rand((rows, 1), generator=g, device="cuda")
        ids = torch.randint(0, vocab, (rows, hot), generator=g, device="cuda")
        noise = 0.3 * torch.randn((rows, hot), generator=g, device="cuda")
        peak = torch.full((rows, vocab), -60.0, device="cuda")
        peak.scatter_reduce_(1, ids, top - steep * rank.log() + noise, "amax")
        v = torch.maximum(v, peak)
    s.logits = v.to(TYPES[case["logits"]])
    s.uniforms = torch.from_numpy(rng.random(rows)).cuda()
    s.mask = None
    if case["density"] > 0:
        words = (vocab + 31) // 32
        allowed = torch.rand((rows, words * 32), generator=g, device="cuda") < case["density"]
        allowed[:, 0] = True
        allowed[:, vocab:] = False
        weight = 1 << torch.arange(32, device="cuda", dtype=torch.int64)
        s.mask = torch.empty((rows, words), dtype=torch.int32, device="cuda")
        for r in range(0, rows, 16):
            packed = (allowed[r:r + 16].view(-1, words, 32).to(torch.int64) * weight).sum(-1)
            s.mask[r:r + 16] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
    s.hist_ids = s.hist_offsets = s.hist_rows = None
    if case["history"]:
        size = rng.integers(0, 2 * case["history"] + 1, rows) if case["mixed"] else np.full(rows, case["history"])
        size[0] = max(1, size[0])
        off = np.concatenate([[0], np.cumsum(size)])
        s.hist_offsets = torch.from_numpy(off.astype(np.int32)).cuda()
        # text repeats ids: a power of a uniform number, then scattered over the vocabulary
        ids = (np.minimum(np.exp(rng.random(off[-1]) * math.log(vocab)), vocab - 1).astype(np.int64) * 7919) % vocab
        s.hist_ids = torch.from_numpy(ids.astype(np.int32)).cuda()
        s.hist_rows = torch.from_numpy(np.repeat(np.arange(rows), size)).cuda()
    p = np.zeros(rows, dtype=PARAMS)
    for name, key in (("temperature", "temperature"), ("top_p", "top_p"), ("min_p", "min_p"), ("top_k", "top_k"),
                      ("repetition_penalty", "repetition"), ("presence_penalty", "presence"), ("frequency_penalty", "frequency")):
        p[name] = case[key]
    if case["mixed"]:
        pick = lambda values: np.array([values[i] for i in rng.integers(0, len(values), rows)])  # noqa: E731
        p["temperature"] = pick([0.0, 0.7, case["temperature"], 1.2])
        p["top_k"] = pick([0, 1, 40, case["top_k"]])
        p["top_p"] = pick([1.0, 0.8, case["top_p"]])
        p["min_p"] = pick([0.0, case["min_p"]])
        p["repetition_penalty"] = pick([1.0, case["repetition"]])
    s.host_params = p
    s.row_params = torch.from_numpy(p.view(np.uint8).reshape(rows, -1).copy()).cuda() if case["mixed"] else None
    # the same as columns, for the plain form
    column = lambda name: torch.from_numpy(p[name].astype(np.float64)).cuda()[:, None]  # noqa: E731
    s.columns = {name: column(name) for name in PARAMS.names}


# ------------------------------------------------------------------ runs --

def run(state):
    if own:
        return _own_project(state) if state.case["kind"] == "project" else _own_sample(state)
    return _plain_project(state) if state.case["kind"] == "project" else _plain_sample(state)


_handle = None


def _sampler():
    global _handle
    if _handle is None:
        from shared_amd import Sampler
        _handle = Sampler(0)  # a program keeps one
    return _handle


def _own_project(s):
    from shared_amd import Adapters
    c = s.case
    return _sampler().project(s.x, s.weight, adapters=Adapters(s.a, s.b, scales=s.scales, ranks=s.ranks),
                              row_adapter=s.row_adapter, softcap=c["softcap"], out_dtype=TYPES[c["y"]])


def _own_sample(s):
    from shared_amd import FilterParams
    p = s.host_params[0]
    params = FilterParams(**{name: p[name].item() for name in PARAMS.names}) if s.row_params is None else None
    r = _sampler().sample_filtered(s.logits, uniforms=s.uniforms, params=params, row_params=s.row_params, mask=s.mask,
                                   hist_ids=s.hist_ids, hist_offsets=s.hist_offsets, full=True)
    return {"ids": r["ids"], "probs": r["probs"], "counts": r["counts"]}


def _plain_project(s):
    c = s.case
    n, rank, dim = s.a.shape
    x = s.x.float()
    y = x @ s.weight.float().T
    h = (x @ s.a.view(n * rank, dim).float().T).view(-1, n, rank)
    pool = torch.arange(n, device="cuda")
    chosen = (s.row_adapter[:, None] == pool) * s.scales
    used = torch.arange(rank, device="cuda") < s.ranks[:, None]
    h = torch.where(used, h, 0.0) * chosen[:, :, None]
    y += h.view(-1, n * rank) @ s.b.permute(0, 2, 1).reshape(n * rank, -1).float()
    if c["softcap"]:
        y = c["softcap"] * torch.tanh(y / c["softcap"])
    return y.to(TYPES[c["y"]])


def _plain_sample(s):
    c, col = s.case, s.columns
    rows, vocab = s.logits.shape
    v = s.logits.to(torch.float32, copy=True)
    if s.hist_ids is not None:
        at = s.hist_rows * vocab + s.hist_ids
        count = torch.zeros(rows * vocab, device="cuda").scatter_add_(0, at, torch.ones(at.numel(), device="cuda"))[at]
        d = v.view(-1)[at].double()
        p = {name: x[s.hist_rows, 0] for name, x in col.items()}
        d = torch.where(d > 0, d / p["repetition_penalty"], d * p["repetition_penalty"])
        d = d - p["frequency_penalty"] * count.double() - p["presence_penalty"]
        v.view(-1)[at] = d.float()  # an id's repeats write the same value
    if s.mask is not None:
        bits = (s.mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        v = torch.where(bits.view(rows, -1)[:, :vocab] > 0, v, -math.inf)
    greedy = col["temperature"] <= 0
    top = v.max(1, keepdim=True).values
    w = torch.exp((v.double() - top.double()) / torch.where(greedy, 1.0, col["temperature"]))
    v, order = torch.sort(v, dim=1, descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(col["top_k"] > 0, col["top_k"], float(vocab))
    k = torch.where(greedy, 1.0, k)
    keep = (rank < k) & (v > -math.inf)
    ws = torch.where(keep, w.gather(1, order), 0.0)
    mass = ws.cumsum(1)
    keep &= (col["top_p"] >= 1) | (rank == 0) | (mass - ws < col["top_p"] * mass[:, -1:])
    keep &= greedy | (ws >= col["min_p"])
    counts = keep.sum(1)
    w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0.0)
    mass = w.cumsum(1)
    total = mass[:, -1:]
    ids = (mass <= s.uniforms[:, None] * total).sum(1, keepdim=True).clamp(max=vocab - 1)
    probs = w.gather(1, ids) / total
    return {"ids": ids[:, 0].to(torch.int32), "probs": probs[:, 0], "counts": counts.to(torch.int32)}


def work(case):
    if case["kind"] == "project":
        rows, dim, out, rank = (case[k] for k in ("rows", "dim", "out", "rank"))
        users, used = _users(case)
        size = {"f32": 4, "bf16": 2}
        return {"bytes": 2 * out * dim + 2 * used * rank * (dim + out) + rows * (size[case["x"]] * dim + size[case["y"]] * out + 4),
                "flops": 2 * rows * dim * out + 2 * users * rank * (dim + out)}
    row = case["vocab"] * (4 if case["logits"] == "f32" else 2) + 24
    row += 4 * ((case["vocab"] + 31) // 32) if case["density"] > 0 else 0
    return {"bytes": case["rows"] * (row + 4 * case["history"]), "flops": 0}


# ------------------------------------------------- the definitions, 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_project(s) if case["kind"] == "project" else _exact_sample(s)


def _exact_project(s):
    y = torch.empty((s.x.shape[0], s.weight.shape[0]), dtype=torch.float64, device="cuda")
    x = s.x.to(torch.float64)
    for at in range(0, s.weight.shape[0], 16384):
        y[:, at:at + 16384] = x @ s.weight[at:at + 16384].to(torch.float64).T
    which = s.row_adapter.cpu().numpy()
    for n in np.unique(which[which >= 0]):
        r = int(s.ranks[n])
        rows = torch.from_numpy(np.nonzero(which == n)[0]).cuda()
        h = x[rows] @ s.a[n, :r].to(torch.float64).T
        y[rows] += float(s.scales[n]) * (h @ s.b[n, :, :r].to(torch.float64).T)
    cap = s.case["softcap"]
    return torch.tanh(y / cap) * cap if cap else y


def _exact_sample(s):
    rows, vocab = s.logits.shape
    u = s.uniforms.cpu().numpy()
    words = None if s.mask is None else s.mask.cpu().numpy().view(np.uint32)
    off = None if s.hist_ids is None else s.hist_offsets.cpu().numpy()
    hist = None if s.hist_ids is None else s.hist_ids.cpu().numpy()
    ids, probs, counts = np.zeros(rows, np.int32), np.zeros(rows), np.zeros(rows, np.int32)
    for r in range(rows):
        p = s.host_params[r]
        v = s.logits[r].to(torch.float64).cpu().numpy()
        if hist is not None:
            seen, times = np.unique(hist[off[r]:off[r + 1]], return_counts=True)
            old = v[seen]
            new = np.where(old > 0, old / p["repetition_penalty"], old * p["repetition_penalty"])
            new = new - p["frequency_penalty"] * times - p["presence_penalty"]
            v[seen] = new.astype(np.float32)  # a penalized value is one of 32 bits again, by definition
        if words is not None:
            v[np.unpackbits(words[r].view(np.uint8), bitorder="little")[:vocab] == 0] = -np.inf
        order = np.argsort(-v, kind="stable")
        if p["temperature"] <= 0:
            ids[r], probs[r], counts[r] = order[0], 1.0, 1
            continue
        w = np.exp((v - v[order[0]]) / p["temperature"])
        n = int((v > -np.inf).sum())
        n = min(n, int(p["top_k"])) if p["top_k"] > 0 else n
        mass = np.cumsum(w[order[:n]])
        if p["top_p"] < 1:
            n = min(n, 1 + int(np.searchsorted(mass, p["top_p"] * mass[-1], side="left")))
        n = min(n, int((w[order[:n]] >= p["min_p"]).sum()))
        kept = np.sort(order[:n])
        mass = np.cumsum(w[kept])
        at = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), n - 1)
        ids[r], probs[r], counts[r] = kept[at], w[kept[at]] / mass[-1], n
    return {"ids": torch.from_numpy(ids), "probs": torch.from_numpy(probs), "counts": torch.from_numpy(counts)}
