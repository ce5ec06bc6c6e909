"""Cases of the serving operators: per-request low-rank adapters, draws from given random numbers, and the
log-probabilities of given tokens.

A case is one call of an operator on the shapes of a serving step: widths of synth.TINY and synth.THREE_B and widths
between them, one decoded token to a packed prefill chunk of 4096 rows, the 65,536-token vocabulary and odd ones.
`own` chooses between the plain form (torch) and the framework's entry points (include/rsv_hip.h).
"""
import ctypes
import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

WIDTHS = (768, 1024, 1536, 2048, 2560)
VOCAB = 65536
IGNORED = -1  # a row of the log-probabilities that asks for none (0xFFFFFFFF)


def listed():
    return [
        # one token of one session on the small model, one square projection: the smallest call, latency
        dict(name="adapters_1", kind="adapters", c=768, k=1, n=1, jobs=1, rows=1, requests=1, pool=4, rank=8,
             x="f32", y="f32", epilogue=0),
        # a decode step of 8 sessions through ffn.key: relu^2 behind the sum, fp16 out for the next product
        dict(name="adapters_8_ffn_key", kind="adapters", c=2560, k=1, n=4, jobs=1, rows=8, requests=8, pool=8, rank=16,
             x="f16", y="f32", epilogue=3),
        # a decode step of 64 sessions with 48 adapters, r/k/v in one call
        dict(name="adapters_64_rkv", kind="adapters", c=2560, k=1, n=1, jobs=3, rows=64, requests=64, pool=48, rank=16,
             x="f16", y="f32", epilogue=0),
        # five prompts of odd lengths packed, ffn.value: the long sum
        dict(name="adapters_517_ffn_value", kind="adapters", c=2560, k=4, n=1, jobs=1, rows=517, requests=5, pool=8,
             rank=32, x="f16", y="f32", epilogue=0),
        # a full packed prefill chunk, r/k/v in one call
        dict(name="adapters_4096_rkv", kind="adapters", c=2560, k=1, n=1, jobs=3, rows=4096, requests=24, pool=12,
             rank=32, x="f16", y="f32", epilogue=0),
        # one session's next token: latency
        dict(name="draw_1", kind="draw", rows=1, n=VOCAB, filters="top_p", logits="f32", spread="peaked"),
        # a step of 8 sessions on an odd vocabulary, fp16 logits (many ties)
        dict(name="draw_8_odd", kind="draw", rows=8, n=65529, filters="top_k", logits="f16", spread="peaked"),
        # a step of 64 sessions, each with settings of its own, greedy ones and grammar masks among them
        dict(name="draw_64_mixed", kind="draw", rows=64, n=VOCAB, filters="mixed", logits="f32", spread="mixed"),
        # 256 samples at temperature 1 with nothing cut: every token counts
        dict(name="draw_256_plain", kind="draw", rows=256, n=VOCAB, filters="none", logits="f32", spread="flat"),
        # the chosen tokens of a decode step of 8 sessions
        dict(name="logprobs_8", kind="logprobs", rows=8, n=VOCAB, logits="f32", spread="peaked"),
        # a short prompt scored, fp16 logits of an odd vocabulary (rows that start at odd halves)
        dict(name="logprobs_100_odd", kind="logprobs", rows=100, n=65529, logits="f16", spread="peaked"),
        # a long prompt scored
        dict(name="logprobs_2048", kind="logprobs", rows=2048, n=VOCAB, logits="f32", spread="mixed"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["adapters", "adapters", "draw", "draw", "logprobs"])
    if kind == "adapters":
        k, n, jobs = rng.choice([(1, 1, 1), (1, 1, 2), (1, 1, 3), (1, 4, 1), (4, 1, 1)])
        rows = _log_int(rng, 1, 4096)
        requests = rows if rows <= 64 else _log_int(rng, 1, 64)  # a decode step, or a packed chunk
        return dict(kind=kind, c=rng.choice(WIDTHS), k=k, n=n, jobs=jobs, rows=rows, requests=requests,
                    pool=_log_int(rng, 1, 64), rank=rng.choice([8, 16, 24, 32, 64, 128]), x=rng.choice(["f16", "f32"]),
                    y=rng.choice(["f32", "f32", "f16"]), epilogue=3 if n == 4 else 0)
    n = rng.choice([VOCAB, VOCAB, 65529, 131072, _log_int(rng, 1000, 131072)])
    rows = min(_log_int(rng, 1, 256 if kind == "draw" else 2048), (256 if kind == "draw" else 2048) * VOCAB // n)
    more = dict(filters=rng.choice(["none", "top_p", "top_k", "min_p", "mixed"])) if kind == "draw" else {}
    return dict(kind=kind, rows=rows, n=n, logits=rng.choice(["f32", "f32", "f16"]),
                spread=rng.choice(["flat", "peaked", "mixed"]), **more)


# ---------------------------------------------------------------- inputs
def _requests(case):
    """(rows of each request, its adapter or -1): fixed by the case.  One request in eight has no adapter."""
    rows, q = case["rows"], case["requests"]
    rng = random.Random(rows * 1009 + q)
    part = [rng.uniform(0.3, 1.0) for _ in range(q)]
    lens = [1 + int((rows - q) * p / sum(part)) for p in part]
    lens[0] += rows - sum(lens)
    order = rng.sample(range(case["pool"]), case["pool"])
    return lens, [-1 if i % 8 == 7 else order[i % case["pool"]] for i in range(q)]


def _ranks(case):
    """An adapter's own rank: the pool's, or for one in four half of it."""
    return [case["rank"] // 2 if a % 4 == 3 else case["rank"] for a in range(case["pool"])]


_TYPES = {"f32": torch.float32, "f16": torch.float16}


class _Gen:
    """Seeded values on the GPU, left where `place` puts them."""

    def __init__(self, seed, place):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(seed)
        self.place = place

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")

    def ints(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device="cuda")

    def logits(self, case):
        """Rows as a head leaves them.  flat: N(0, 1); peaked: N(0, 2.5^2) with 40 likely tokens above it; mixed: the
        two in turn, and every fifth row masked down to about 200 tokens, as a grammar does."""
        rows, n = case["rows"], case["n"]
        l = self.normal(rows, n)
        row = torch.arange(rows, device="cuda")
        peaked = torch.full((rows,), case["spread"] == "peaked", device="cuda")
        if case["spread"] == "mixed":
            peaked = row % 2 == 1
        l.mul_(torch.where(peaked, 2.5, 1.0)[:, None])
        likely = self.ints(n, rows, 40)
        l.scatter_add_(1, likely, (6.0 + 6.0 * self.uniform(rows, 40)) * peaked[:, None])
        if case["spread"] == "mixed":
            for r in range(4, rows, 5):
                l[r][self.uniform(n) > 200.0 / n] = -math.inf
                l[r, likely[r, 0]] = 1.0
        return self.place(l.to(_TYPES[case["logits"]]))


def _filters(case, rows):
    """Temperature, top-k, top-p and min-p of each row, as the host holds them."""
    kinds = {"none": (1.0, 0, 1.0, 0.0), "top_p": (1.0, 0, 0.9, 0.0), "top_k": (0.8, 50, 0.95, 0.0),
             "min_p": (1.3, 0, 1.0, 0.05), "greedy": (0.0, 0, 1.0, 0.0)}
    names = ["none", "top_p", "top_k", "min_p"] if case["filters"] == "mixed" else [case["filters"]]
    got = [kinds[names[r % len(names)]] for r in range(rows)]
    if case["filters"] == "mixed":
        got = [kinds["greedy"] if r % 16 == 5 else v for r, v in enumerate(got)]
    return got


class _State:
    """What a case's pass needs: its tensors, and for the framework's calls the prepared calls and their outputs."""

    def __init__(self, case):
        self.case, self.steps, self.keep, self.out = case, [], [], None


def _inputs(case, seed, place=lambda t: t):
    g, s = _Gen(seed, place), _State(case)
    if case["kind"] == "adapters":
        c, rows, pool, rank = case["c"], case["rows"], case["pool"], case["rank"]
        s.k, s.n = case["k"] * c, case["n"] * c
        lens, ids = _requests(case)
        s.ids = place(torch.tensor(np.repeat(ids, lens).astype(np.int32), device="cuda"))
        s.ranks = place(torch.tensor(_ranks(case), dtype=torch.int32, device="cuda"))
        s.scale = place(0.5 + g.uniform(pool))
        s.jobs = [dict(a=place(g.normal(pool, rank, s.k, std=s.k ** -0.5).half()),
                       b=place(g.normal(pool, s.n, rank, std=0.3 * rank ** -0.5).half()),
                       x=place(g.normal(rows, s.k).to(_TYPES[case["x"]])),
                       y=place(g.normal(rows, s.n).to(_TYPES[case["y"]]))) for _ in range(case["jobs"])]
        return s
    s.logits = g.logits(case)
    rows, n = case["rows"], case["n"]
    if case["kind"] == "draw":
        rows4 = np.zeros((rows, 4), np.float32)
        for r, (t, k, p, m) in enumerate(_filters(case, rows)):
            rows4[r] = t, np.uint32(k).view(np.float32), p, m
        s.filters = place(torch.tensor(rows4, device="cuda"))
        s.u = place(g.uniform(rows))
    else:
        top = s.logits.float().topk(min(50, n), 1).indices
        likely = top.gather(1, g.ints(top.shape[1], rows, 1))[:, 0]
        tok = torch.where(g.uniform(rows) < 0.8, likely, g.ints(n, rows)).int()
        tok[127::128] = IGNORED  # a prompt's last position has no next token
        s.tokens = place(tok)
    return s


def _out_type(case):
    """The type the next product takes: fp16 behind ffn.key, otherwise the sum's own."""
    return "f16" if case["epilogue"] == 3 else case["y"]


# ---------------------------------------------------------------- the plain form
def _adapters_plain(s):
    """Every row against every adapter of the pool, its own kept: no gather of weights by row, no loop over adapters."""
    case, pool, rank = s.case, s.case["pool"], s.case["rank"]
    place = torch.arange(pool * rank, device="cuda")
    mine = (place // rank == s.ids[:, None]) & (place % rank < s.ranks[place // rank])
    weight = torch.where(mine, s.scale[place // rank], 0.0)
    def one(j):
        h = (j["x"].float() @ j["a"].float().view(pool * rank, s.k).T) * weight
        z = j["y"].float() + h @ j["b"].float().transpose(1, 2).reshape(pool * rank, s.n)
        return (torch.relu(z).square() if case["epilogue"] == 3 else z).to(_TYPES[_out_type(case)])
    return list(map(one, s.jobs))


def _draw_plain(s):
    n = s.case["n"]
    t, p, m = (s.filters[:, i, None].double() for i in (0, 2, 3))
    top_k = s.filters[:, 1, None].contiguous().view(torch.int32)
    top_k = torch.where(top_k == 0, n, top_k)
    greedy = ~(t > 0)
    l = s.logits.double()
    z = (l - l.amax(1, keepdim=True)) / torch.where(greedy, 1.0, t)
    e = z.exp()
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    es, at = e.gather(1, order), torch.arange(n, device="cuda")
    es = torch.where((at < top_k) & (es >= m), es, 0.0)
    before = es.cumsum(1) - es
    keep = (es > 0) & ((before < p * es.sum(1, keepdim=True)) | (p >= 1) | (at == 0)) & (~greedy | (at == 0))
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    sums = torch.where(kept, e, 0.0).cumsum(1)
    tok = (sums <= s.u[:, None].double() * sums[:, -1:]).sum(1, keepdim=True)
    tok = torch.minimum(tok, torch.where(kept, at, 0).amax(1, keepdim=True))
    return dict(token=tok[:, 0].int(), logp=(z.gather(1, tok) - sums[:, -1:].log())[:, 0].float())


def _logprobs_plain(s):
    l = s.logits.float()
    asked = (s.tokens >= 0) & (s.tokens < s.case["n"])
    tok = torch.where(asked, s.tokens, 0)[:, None].long()
    top, own_l = l.amax(1, keepdim=True), l.gather(1, tok)
    logp = (own_l - top) - (l - top).exp().sum(1, keepdim=True).log()
    at = torch.arange(s.case["n"], device="cuda")
    rank = ((l > own_l) | ((l == own_l) & (at < tok))).sum(1)
    return dict(logp=torch.where(asked, logp[:, 0], 0.0), rank=torch.where(asked, rank, 0).int())


# ---------------------------------------------------------------- the framework's calls
@functools.lru_cache(None)
def _rsv():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-rsv_amd"))
    import rsv
    return rsv, rsv.Backend(0)


class _Mem:
    """A tensor of the backend, freed when nothing refers to it; torch views it in place."""

    def __init__(self, n, dtype):
        rsv, self.be = _rsv()
        code = {torch.float32: rsv.F32, torch.float16: rsv.F16, torch.int32: rsv.U32}[dtype]
        self.id, self.free = self.be.tensor(n=n, dtype=code), rsv.hip_lib().rsv_tensor_free
        p = ctypes.c_void_p()
        self.be.call("rsv_tensor_ptr", self.id, ctypes.byref(p))
        kind = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4"}[dtype]
        self.__cuda_array_interface__ = dict(shape=(n,), typestr=kind, data=(p.value, False), version=2, strides=None)

    def __del__(self):
        self.free(self.be.ctx, self.id)


class _Device:
    """Puts tensors into the backend's memory: torch's views of them, and their ids."""

    def __init__(self):
        self.mems = {}

    def new(self, shape, dtype):
        mem = _Mem(math.prod(shape), dtype)
        t = torch.as_tensor(mem, device="cuda").view(shape)
        self.mems[t.data_ptr()] = mem
        return t

    def put(self, t):
        return self.new(t.shape, t.dtype).copy_(t)

    def id(self, t):
        return self.mems[t.data_ptr()].id


def _calls(s, d):
    rsv, be = _rsv()
    lib, case, rows = rsv.hip_lib(), s.case, s.case["rows"]

    def op(name, *args):
        s.keep.append(args)
        s.steps.append(functools.partial(getattr(lib, name), be.ctx, *args))

    if case["kind"] == "adapters":
        outs = [d.new((rows, s.n), _TYPES[_out_type(case)]) for _ in s.jobs]
        jobs = (rsv.AdapterJob * len(s.jobs))(*[
            rsv.AdapterJob(d.id(j["a"]), d.id(j["b"]), s.n, s.k, d.id(j["x"]), d.id(j["y"]), d.id(o), case["epilogue"])
            for j, o in zip(s.jobs, outs)])
        work = d.new((max(1, lib.rsv_adapter_work(jobs, len(jobs), case["rank"], rows)),), torch.float32)
        op("rsv_adapter_multi", jobs, len(jobs), d.id(s.ids), d.id(s.scale), d.id(s.ranks), case["pool"], case["rank"],
           rows, d.id(work))
        s.out = outs
    else:
        n, logp = case["n"], d.new((rows,), torch.float32)
        work, whole = d.new((max(1, lib.rsv_logits_work(n, rows)),), torch.float32), d.new((rows,), torch.int32)
        if case["kind"] == "draw":
            op("rsv_sample_rand_batch", d.id(s.logits), d.id(whole), n, d.id(s.filters), d.id(s.u), d.id(logp),
               d.id(work), rows)
            s.out = dict(token=whole, logp=logp)
        else:
            op("rsv_token_logprobs", d.id(s.logits), d.id(s.tokens), n, d.id(logp), d.id(whole), d.id(work), rows)
            s.out = dict(logp=logp, rank=whole)
    s.keep.append((d, work))
    return s


def prepare(case, seed):
    if own:
        d = _Device()
        s = _calls(_inputs(case, seed, d.put), d)
    else:
        s = _inputs(case, seed)
    torch.cuda.synchronize()
    return s


def run(state):
    if own:
        for step in state.steps:
            if step():
                raise RuntimeError(_rsv()[0].hip_lib().rsv_last_error().decode())
        return state.out
    return {"adapters": _adapters_plain, "draw": _draw_plain, "logprobs": _logprobs_plain}[state.case["kind"]](state)


# ---------------------------------------------------------------- work
_BYTES = {"f32": 4, "f16": 2}


def work(case):
    if case["kind"] == "adapters":
        lens, ids = _requests(case)
        ranks, rows, jobs = _ranks(case), case["rows"], case["jobs"]
        k, n = case["k"] * case["c"], case["n"] * case["c"]
        weights = sum(ranks[a] for a in set(ids) if a >= 0) * (k + n) * 2
        moved = rows * (k * _BYTES[case["x"]] + n * (_BYTES[case["y"]] + _BYTES[_out_type(case)]))
        return dict(bytes=jobs * (weights + moved),
                    flops=jobs * sum(2 * m * ranks[a] * (k + n) for m, a in zip(lens, ids) if a >= 0))
    values = case["rows"] * case["n"]
    return dict(bytes=values * _BYTES[case["logits"]] + case["rows"] * 32, flops=4 * values)


# ---------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "adapters":
        outs, ids, ranks = [], s.ids.long(), _ranks(case)
        for j in s.jobs:
            z = j["y"].double()
            for a in sorted(set(ids.tolist()) - {-1}):
                rows = torch.nonzero(ids == a)[:, 0]
                h = j["x"][rows].double() @ j["a"][a, :ranks[a]].double().T.contiguous()
                z[rows] += s.scale[a].double() * (h @ j["b"][a, :, :ranks[a]].double().T.contiguous())
            outs.append(z.clamp_min(0) ** 2 if case["epilogue"] == 3 else z)
        return outs
    l = s.logits.double().cpu().numpy()
    if case["kind"] == "logprobs":
        logp = np.zeros(case["rows"])
        for r, tok in enumerate(s.tokens.tolist()):
            if tok >= 0:
                top = l[r].max()
                logp[r] = l[r, tok] - top - math.log(np.exp(l[r] - top).sum())
        return dict(logp=logp, rank=None)
    logp = np.zeros(case["rows"])
    for r, ((t, k, p, m), u) in enumerate(zip(_filters(case, case["rows"]), s.u.tolist())):
        if t <= 0:
            continue  # the largest logit, drawn with certainty
        p, m, t = float(np.float32(p)), float(np.float32(m)), float(np.float32(t))
        order = np.argsort(-l[r], kind="stable")[:k or None]
        z = (l[r, order] - l[r, order[0]]) / t
        e = np.exp(z)
        e = e[e >= m]
        if p < 1:
            e = e[:max(1, np.count_nonzero(np.cumsum(e) - e < p * e.sum()))]
        inside = np.sort(order[:len(e)])
        at = np.cumsum(np.exp((l[r, inside] - l[r, order[0]]) / t))
        tok = inside[min(len(inside) - 1, np.searchsorted(at, u * at[-1], side="right"))]
        logp[r] = (l[r, tok] - l[r, order[0]]) / t - math.log(at[-1])
    return dict(token=None, logp=logp)
