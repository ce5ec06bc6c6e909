"""Per-request adapters, draws from given random numbers and token
log-probabilities (rsv_adapter_multi, rsv_sample_rand_batch,
rsv_token_logprobs) against their formulas in float64, through the C-ABI."""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF
U = 2.0 ** -24  # half a step of fp32, relative
UH = 2.0 ** -11  # of fp16


@pytest.fixture(scope="module")
def be():
    import rsv
    b = rsv.Backend(0)
    yield b
    b.close()


@pytest.fixture()
def tens(be):
    """Tensors of one test, freed behind it."""
    import rsv
    made = []

    class T:
        def __call__(self, data=None, n=None, dtype=rsv.F32):
            made.append(be.tensor(data, n, dtype))
            return made[-1]

        def f16(self, a):
            return self(np.asarray(a, np.float32), dtype=rsv.F16)

        def u32(self, a):
            return self(np.asarray(a, np.uint32), dtype=rsv.U32)

        def real(self, a, kind):
            return self.f16(a) if kind == "f16" else self(a)
    yield T()
    for t in made:
        be.call("rsv_tensor_free", t)


def kind_of(name):
    import rsv
    return {"f32": rsv.F32, "f16": rsv.F16}[name]


# ------------------------------------------------------------- adapters
class Adapters:
    """One call's operands, on the host and on the device."""

    def __init__(self, tens, rng, rows, na, rank, shapes, x="f32", y="f32", out="f32", epi=0, ranks=None, ids=None,
                 inplace=False):
        import rsv
        self.rows, self.na, self.rank, self.epi, self.out_kind = rows, na, rank, epi, out
        self.ids = rng.integers(0, na + 1, rows).astype(np.uint32) if ids is None else np.asarray(ids, np.uint32)
        self.ids = np.where(self.ids == na, np.uint32(NONE), self.ids) if ids is None else self.ids
        self.ranks = ranks
        self.scale = rng.uniform(-2, 2, na).astype(np.float32)
        half = lambda a: np.asarray(a, np.float16).astype(np.float32)  # noqa: E731
        self.host, jobs = [], []
        for k, n in shapes:
            a = half(rng.standard_normal((na, rank, k)) * k ** -0.5)
            b = half(rng.standard_normal((na, n, rank)) * rank ** -0.5)
            xs, ys = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
            xs, ys = (half(xs) if x == "f16" else xs), (half(ys) if y == "f16" else ys)
            self.host.append([a, b, xs, ys])
        self.tens, self.x_kind, self.y_kind, self.inplace, self.shapes = tens, x, y, inplace, shapes

    def upload(self):
        import rsv
        t = self.tens
        self.t_ids, self.t_scale = t.u32(self.ids), t(self.scale)
        self.t_ranks = NONE if self.ranks is None else t.u32(self.ranks)
        self.t_out, jobs = [], []
        for (a, b, xs, ys), (k, n) in zip(self.host, self.shapes):
            ty = t.real(ys, self.y_kind)
            to = ty if self.inplace else t(n=self.rows * n, dtype=kind_of(self.out_kind))
            self.t_out.append(to)
            jobs.append(rsv.AdapterJob(t.f16(a), t.f16(b), n, k, t.real(xs, self.x_kind), ty, to, self.epi))
        self.jobs = (rsv.AdapterJob * len(jobs))(*jobs)
        self.work = t(n=rsv.hip_lib().rsv_adapter_work(self.jobs, len(jobs), self.rank, self.rows))
        return self

    def call(self, be):
        be.call("rsv_adapter_multi", self.jobs, len(self.jobs), self.t_ids, self.t_scale, self.t_ranks, self.na,
                self.rank, self.rows, self.work)

    def get(self, be):
        return [be.get(t, self.rows * n, kind_of(self.out_kind)).reshape(self.rows, n)
                for t, (k, n) in zip(self.t_out, self.shapes)]

    def want(self):
        """Each job's result in float64, and how far fp32 sums in any order may be from it: a sum of N products in any
        order is off by at most N half steps of the sum of their sizes."""
        res = []
        for (a, b, xs, ys), (k, n) in zip(self.host, self.shapes):
            z, off = ys.astype(np.float64), np.abs(ys).astype(np.float64) * 2 * U
            for i in np.unique(self.ids[self.ids < self.na]):
                R = self.rank if self.ranks is None else min(int(self.ranks[i]), self.rank)
                at = np.nonzero(self.ids == i)[0]
                A, B = a[i, :R].astype(np.float64), b[i, :, :R].astype(np.float64)
                X, s = xs[at].astype(np.float64), float(self.scale[i])
                z[at] += s * ((X @ A.T) @ B.T)
                off[at] += (k + R + 8) * U * abs(s) * ((np.abs(X) @ np.abs(A).T) @ np.abs(B).T)
            if self.epi == 3:
                p = np.maximum(z, 0)
                z, off = p * p, (2 * p + off) * off + 2 * U * p * p
            if self.out_kind == "f16":
                off = off * (1 + UH) + UH * np.abs(z) + 2.0 ** -25
            res.append((z, off))
        return res

    def check(self, be):
        for got, (z, off) in zip(self.get(be), self.want()):
            bad = ~(np.abs(got - z) <= off)
            assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], z[bad][:4])
            # roundings of a sum wander: their norm is about the root of their number, not the number
            depth = max(k for k, _ in self.shapes) + self.rank
            lim = off * 6 / math.sqrt(depth) + 2 * U * np.abs(z) + (UH * np.abs(z) + 2.0 ** -25 if self.out_kind == "f16" else 0)
            assert np.linalg.norm(got - z) <= np.linalg.norm(lim)


SHAPES = [
    # rows, adapters, rank, [(k, n)]
    (1, 1, 8, [(8, 8)]),
    (1, 4, 16, [(768, 768)]),
    (3, 2, 24, [(136, 72)]),
    (17, 5, 8, [(776, 1000)]),
    (64, 48, 16, [(512, 640), (512, 640), (512, 640)]),
    (65, 3, 128, [(264, 520), (1032, 8)]),
    (130, 130, 40, [(328, 264)]),
    (200, 1, 64, [(2560, 320)]),
    (517, 7, 32, [(640, 136)]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dr%d" % s[:3])
@pytest.mark.parametrize("types", [("f16", "f32", "f32"), ("f32", "f32", "f32"), ("f16", "f16", "f16"), ("f32", "f16", "f32")],
                         ids="-".join)
def test_adapters(be, tens, shape, types):
    rows, na, rank, shapes = shape
    rng = np.random.default_rng(rows * 7 + na + rank)
    c = Adapters(tens, rng, rows, na, rank, shapes, *types, epi=3 if rows % 2 else 0).upload()
    c.call(be)
    c.check(be)


@pytest.mark.parametrize("rows,k,n,rank,na", [(8, 2560, 10240, 16, 8), (5, 10240, 2560, 64, 2), (300, 2560, 2560, 32, 4),
                                              (1, 2560, 2560, 128, 3), (40, 2560, 768, 96, 2)])
@pytest.mark.parametrize("x", ["f16", "f32"])
def test_adapters_model_shapes(be, tens, rows, k, n, rank, na, x):
    rng = np.random.default_rng(rows + k)
    ids = np.repeat(rng.permutation(na + 1), -(-rows // (na + 1)))[:rows]  # requests' rows stand together
    c = Adapters(tens, rng, rows, na, rank, [(k, n)], x, "f32", "f32", ids=np.where(ids == na, NONE, ids)).upload()
    c.call(be)
    c.check(be)


def test_adapters_own_ranks_and_what_lies_past_them(be, tens):
    """Ranks 0, odd ones and past the pool's; rows of a and b past an adapter's rank, and adapters no row uses, hold
    NaN and infinities."""
    rng = np.random.default_rng(5)
    ranks = np.array([0, 1, 3, 8, 13, 31, 32, 1000, 7], np.uint32)
    ids = np.concatenate([np.arange(8), [NONE, 9, 2 ** 31], np.repeat([4, 6], 30), rng.integers(0, 8, 40)])
    for x in ("f16", "f32"):
        c = Adapters(tens, rng, len(ids), 9, 32, [(264, 136)], x, ranks=ranks, ids=ids)
        c.upload()
        a, b = c.host[0][:2]
        for i, r in enumerate(ranks):
            a[i, r:], b[i, :, r:] = np.nan, np.inf
        a[8], b[8] = np.inf, np.nan
        c.jobs[0].a, c.jobs[0].b = tens.f16(a), tens.f16(b)
        c.call(be)
        a[:], b[:] = np.nan_to_num(a, nan=0, posinf=0), np.nan_to_num(b, nan=0, posinf=0)
        c.check(be)
        got = c.get(be)[0]
        bare = (c.ids >= 9) | (c.ids == 0)
        assert np.array_equal(got[bare], c.host[0][3][bare])  # no adapter (or one of rank 0): y's own bits


@pytest.mark.parametrize("rows", [9, 150])
def test_adapters_in_place_and_non_finite_rows(be, tens, rows):
    """out = y; a row with infinities in x or y leaves every other row as it was; scale 0 and NaN act on their own."""
    rng = np.random.default_rng(rows)
    c = Adapters(tens, rng, rows, 4, 16, [(520, 264)], "f16", "f32", inplace=True).upload()
    c.call(be)
    c.check(be)
    clean = c.get(be)[0]
    d = Adapters(tens, np.random.default_rng(rows), rows, 4, 16, [(520, 264)], "f16", "f32")
    d.ids[2], d.ids[5] = 1, NONE
    d.host[0][2][2, 7] = np.inf
    d.host[0][3][5, 3] = np.nan
    d.upload()
    d.call(be)
    got = d.get(be)[0]
    same = np.ones(rows, bool)
    same[[2, 5]] = False
    assert np.array_equal(got[same], clean[same])
    assert not np.isfinite(got[2]).any() and np.isnan(got[5, 3]) and np.isfinite(np.delete(got[5], 3)).all()


@pytest.mark.parametrize("rows", [6, 100])
def test_adapters_large_scale_beside_small_weights(be, tens, rows):
    """scale times h is past fp32's range, their product with b is not: 1e12 * 1e30 * 1e-4."""
    rng = np.random.default_rng(3)
    c = Adapters(tens, rng, rows, 2, 8, [(64, 136)], ranks=[1, 1])
    c.scale[:] = 1e12
    a, b, x, _ = c.host[0]
    a[:], x[:] = 1.0, np.float32(1e30 / 64) * rng.uniform(0.5, 1.0, x.shape).astype(np.float32)
    b[:] = np.float16(1e-4)
    c.upload()
    c.call(be)
    c.check(be)


def test_adapters_far_offsets(be, tens):
    """An adapter whose matrices lie past 2^31 elements of the pool."""
    import rsv
    torch = pytest.importorskip("torch")
    na, rank, k, n, rows = 1040, 128, 16384, 64, 3
    rng = np.random.default_rng(1)
    a = np.asarray(rng.standard_normal((rank, k)) / 128, np.float16)
    b = np.asarray(rng.standard_normal((n, rank)) / 11, np.float16)
    pool_a, pool_b = tens(n=na * rank * k, dtype=rsv.F16), tens(n=na * n * rank, dtype=rsv.F16)
    for t, v, at in ((pool_a, a, (na - 1) * rank * k), (pool_b, b, (na - 1) * n * rank)):
        p = ctypes.c_void_p()
        be.call("rsv_tensor_ptr", t, ctypes.byref(p))
        mem = type("M", (), {"__cuda_array_interface__": dict(shape=(v.size,), typestr="<f2", version=2, strides=None,
                                                              data=(p.value + 2 * at, False))})()
        torch.as_tensor(mem, device="cuda").copy_(torch.from_numpy(v.reshape(-1)))
    torch.cuda.synchronize()
    x = rng.standard_normal((rows, k)).astype(np.float32)
    y = np.zeros((rows, n), np.float32)
    out = tens(n=rows * n)
    jobs = (rsv.AdapterJob * 1)(rsv.AdapterJob(pool_a, pool_b, n, k, tens(x), tens(y), out, 0))
    work = tens(n=rsv.hip_lib().rsv_adapter_work(jobs, 1, rank, rows))
    be.call("rsv_adapter_multi", jobs, 1, tens.u32([na - 1, 0, na - 1]), tens(np.ones(na)), NONE, na, rank, rows, work)
    got = be.get(out, rows * n).reshape(rows, n)
    X, A, B = x.astype(np.float64), a.astype(np.float64), b.astype(np.float64)
    want, off = (X @ A.T) @ B.T, (k + rank + 8) * U * ((np.abs(X) @ np.abs(A).T) @ np.abs(B).T)
    assert (np.abs(got - want)[[0, 2]] <= off[[0, 2]]).all() and (got[1] == 0).all()


def test_adapters_replayed(be, tens):
    """A captured call follows the rows' adapters, the scales and the inputs as they are at each replay, with eager
    calls between the replays."""
    rng = np.random.default_rng(3)
    c = Adapters(tens, rng, 70, 6, 16, [(520, 264), (264, 520)], "f16", "f32").upload()
    c.call(be)  # eager once
    c.check(be)
    be.call("rsv_graph_begin")
    c.call(be)
    be.call("rsv_graph_end")
    for rep in range(3):
        c.ids = rng.integers(0, 7, 70).astype(np.uint32)
        c.scale = rng.uniform(-1, 1, 6).astype(np.float32)
        be.call("rsv_upload_u32", c.t_ids, c.ids.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32)), c.ids.size)
        be.call("rsv_upload", c.t_scale, c.scale.ctypes.data_as(ctypes.POINTER(ctypes.c_float)), c.scale.size)
        be.call("rsv_graph_replay")
        got = c.get(be)
        c.check(be)
        c.call(be)
        for g, e in zip(got, c.get(be)):
            assert np.array_equal(g, e)


def test_adapters_refusals(be, tens):
    import rsv
    rng = np.random.default_rng(0)
    c = Adapters(tens, rng, 70, 2, 16, [(64, 32), (64, 32)], "f16").upload()
    args = lambda **o: [o.get("jobs", c.jobs), o.get("njobs", 2), o.get("ids", c.t_ids), o.get("scale", c.t_scale),  # noqa: E731
                        o.get("ranks", c.t_ranks), o.get("na", 2), o.get("rank", 16), o.get("rows", 70), o.get("work", c.work)]
    def job(i=0, **f):
        js = (rsv.AdapterJob * 2)(*[rsv.AdapterJob(*[getattr(j, n) for n, _ in j._fields_]) for j in c.jobs])
        for n, v in f.items():
            setattr(js[i], n, v)
        return js
    j0, j1 = c.jobs
    for match, bad in [
            ("1..8 jobs", dict(njobs=0)), ("1..8 jobs", dict(njobs=9)), ("1..8 jobs", dict(jobs=None)),
            ("rank 0", dict(rank=0)), ("rank 12", dict(rank=12)), ("rank 136", dict(rank=136)),
            ("rows 0", dict(rows=0)), ("rows 1048577", dict(rows=1048577)), ("needs", dict(rows=71)),
            ("n_adapter 0", dict(na=0)), ("needs", dict(na=3)), ("unknown tensor", dict(ids=9999999)),
            ("unknown tensor", dict(scale=NONE)), ("needs", dict(work=c.t_scale)), ("unknown tensor", dict(work=NONE)),
            ("multiples of 8", dict(jobs=job(n=0))), ("multiples of 8", dict(jobs=job(k=60))),
            ("multiples of 8", dict(jobs=job(n=12))), ("epilogue 2", dict(jobs=job(epilogue=2))),
            ("unknown tensor", dict(jobs=job(a=NONE))), ("dtype", dict(jobs=job(a=j0.y))), ("needs", dict(jobs=job(1, n=40))),
            ("must be F32 or F16", dict(jobs=job(x=c.t_ids))), ("another operand", dict(jobs=job(out=j1.out))),
            ("another operand", dict(jobs=job(out=j1.y))), ("another operand", dict(jobs=job(1, out=j0.x))),
            ("another operand", dict(jobs=job(y=c.work, out=c.t_out[0]), work=c.work))]:
        if match == "another operand" and "work" in bad:
            big = tens(n=1 << 20)
            bad = dict(jobs=job(y=big), work=big)
        with pytest.raises(rsv.RsvError, match=match):
            be.call("rsv_adapter_multi", *args(**bad))
    c.call(be)
    c.check(be)


# ------------------------------------------------------------- draws
def order_of(l):
    """Tokens by logit, larger first, equal ones by index."""
    return np.argsort(-l, kind="stable")


def draw64(l, T, top_k, top_p, min_p, u):
    """(token, logp) of one row by the formula in float64."""
    l = np.where(np.isnan(l), -np.inf, np.asarray(l, np.float64))
    m = l.max()
    if m == -np.inf:
        return NONE, -np.inf
    if not T > 0:
        return int(np.argmax(l)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(l == m, 0.0, np.where(l == -np.inf, -np.inf, (l - m) / np.float64(T)))
    o = order_of(l)[:top_k or None]
    e = np.exp(z[o])
    keep = e >= (min(float(min_p), 1.0) if min_p > 0 else 0.0)
    o, e = o[keep], e[keep]
    if top_p < 1:
        o = o[:max(1, np.count_nonzero(np.cumsum(e) - e < float(top_p) * e.sum()))]
    o = np.sort(o)
    c = np.cumsum(np.exp(z[o]))
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    live = np.nonzero(np.exp(z[o]) > 0)[0]
    tok = o[min(live[-1], np.searchsorted(c, u * c[-1], side="right"))]
    return int(tok), z[tok] - math.log(c[-1])


def filters_of(rows):
    f = np.zeros((len(rows), 4), np.float32)
    for i, (t, k, p, m) in enumerate(rows):
        f[i] = t, np.uint32(k).view(np.float32), p, m
    return f


def run_draw(be, tens, l, filters, u, kind="f32"):
    import rsv
    rows, n = l.shape
    tok, logp = tens(n=rows, dtype=rsv.U32), tens(n=rows)
    work = tens(n=max(1, rsv.hip_lib().rsv_logits_work(n, rows)))
    be.call("rsv_sample_rand_batch", tens.real(l, kind), tok, n, tens(filters_of(filters)), tens(u), logp, work, rows)
    return be.get(tok, rows, rsv.U32), be.get(logp, rows)


def check_draw(be, tens, l, filters, u, kind="f32"):
    l = np.asarray(l, np.float32)
    if kind == "f16":
        l = l.astype(np.float16).astype(np.float32)
    filters = [tuple(np.float32(v) if j != 1 else v for j, v in enumerate(f)) for f in filters]
    u = np.asarray(u, np.float32)
    tok, logp = run_draw(be, tens, l, filters, u, kind)
    for r in range(len(l)):
        want, lp = draw64(l[r], *filters[r], u[r])
        assert tok[r] == want, (r, filters[r], u[r], tok[r], want, l[r][tok[r]] if tok[r] < l.shape[1] else None, l[r][want])
        # fp64 inside, one rounding to fp32; the weights are off by half of 2^-36 of the largest each, either way: root
        # of 65536 times 0.29 times 2^-36 is 1e-9 of a sum that is not less than the largest
        assert logp[r] == lp or abs(logp[r] - lp) <= 2 * U * abs(lp) + 1e-9, (r, logp[r], lp)


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 40, 1.0, 0.0), (1.0, 0, 1.0, 0.1), (0.9, 200, 0.8, 0.02),
           (0.0, 0, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (2.0, 0, 0.3, 0.0), (1.0, 3, 0.999, 0.0)]


@pytest.mark.parametrize("n", [1, 2, 7, 63, 64, 65, 1000, 1024, 4097, 50001, 65529, 65536])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_draw(be, tens, n, kind):
    rng = np.random.default_rng(n)
    rows = 30
    l = rng.standard_normal((rows, n)) * rng.choice([0.0, 1.0, 4.0], (rows, 1))
    l[np.arange(rows), rng.integers(0, n, rows)] += rng.choice([0, 8], rows)
    l[3::5] = np.where(rng.random((6, n)) < 0.9, -np.inf, l[3::5])  # masked rows: some with few or no tokens left
    if n > 4:
        l[4::5] = np.round(l[4::5])  # many equal logits
    check_draw(be, tens, l, [FILTERS[r % 10] for r in range(rows)], rng.random(rows), kind)


@pytest.mark.parametrize("rows,n", [(300, 1500), (1, 131072), (2, 1048576), (70, 70000), (1100, 40)])
def test_draw_sizes(be, tens, rows, n):
    rng = np.random.default_rng(rows)
    l = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
    check_draw(be, tens, l, [FILTERS[r % 10 if rows > 2 else r + 1] for r in range(rows)], rng.random(rows))


@pytest.mark.parametrize("spread", [0.02, 1.0, 3.0, 30.0])
@pytest.mark.parametrize("top_p", [0.05, 0.5, 0.9, 0.999])
def test_draw_nucleus_from_flat_to_peaked(be, tens, spread, top_p):
    rng = np.random.default_rng(int(spread * 100))
    l = rng.standard_normal((6, 65536)) * spread
    f = [(1.0, 0, top_p, 0.0), (0.5, 0, top_p, 0.0), (1.0, 1000, top_p, 0.0), (1.0, 0, top_p, 1e-3), (5.0, 0, top_p, 0.0),
         (1.0, 30000, top_p, 1e-6)]
    check_draw(be, tens, l, f, rng.random(6))
    check_draw(be, tens, l, f, rng.random(6), "f16")


@pytest.mark.parametrize("count", [1, 2, 63, 65, 128, 255, 256, 257, 600, 1024, 1025, 5000])
@pytest.mark.parametrize("n", [20001, 70001])
def test_draw_among_few_tokens(be, tens, count, n):
    """All weight on `count` tokens anywhere in a row, half of them in groups of equal logits; rows that do not start
    at a 16-byte border."""
    rng = np.random.default_rng(count * 7 + n)
    f = [(1.0, 0, 0.9, 0.0), (0.7, count // 2 + 1, 0.8, 0.0), (1.0, count, 1.0, 0.0), (1.0, 0, 0.95, 0.2),
         (1.0, count + 3, 0.999, 0.0), (2.0, 0, 1.0, 0.5), (1.0, max(1, count // 3), 0.6, 0.3)]
    l = rng.standard_normal((len(f), n)) - 40.0
    for r in range(len(f)):
        at = rng.permutation(n)[:count]
        v = rng.standard_normal(count) * 0.4
        v[::2] = np.round(v[::2] * 4) / 4
        l[r, at] = v
    check_draw(be, tens, l, f, rng.random(len(f)))
    check_draw(be, tens, l, f, rng.random(len(f)), "f16")


def test_draw_every_token_by_its_share(be, tens):
    """u over a grid draws each token as often as its probability says, cut at the grid's steps."""
    l = np.log(np.array([0.5, 0.125, 0.25, 0.0625, 0.0625], np.float64))
    u = (np.arange(256) + 0.5) / 256
    tok, _ = run_draw(be, tens, np.tile(l.astype(np.float32), (256, 1)), [(1.0, 0, 1.0, 0.0)] * 256, u)
    assert np.bincount(tok, minlength=5).tolist() == [128, 32, 64, 16, 16]


def test_draw_ties_are_cut_by_index(be, tens):
    """Equal logits: top-k and top-p take the lower indexes; sums are whole numbers, so the borders are exact."""
    n, u = 4096, [0.0, 0.25, 0.49999997, 0.5, 0.99999994, 1.0]
    l = np.zeros((6, n))
    check_draw(be, tens, l, [(1.0, 0, 1.0, 0.0)] * 6, u)
    check_draw(be, tens, l, [(1.0, 100, 1.0, 0.0)] * 6, u)
    check_draw(be, tens, l, [(1.0, 0, 0.5, 0.0)] * 6, u)
    check_draw(be, tens, l, [(1.0, 100, 0.5, 1.0)] * 6, u)
    l[:, 1000:1003] = 2.0
    check_draw(be, tens, l, [(1.0, 2, 1.0, 0.0)] * 6, u)
    check_draw(be, tens, l, [(1.0, 50, 0.97, 0.0)] * 6, u)
    check_draw(be, tens, l, [(1.0, 0, 1.0, 1.0)] * 6, u)


def test_draw_non_finite(be, tens):
    inf, nan = np.inf, np.nan
    l = np.array([[-inf] * 4, [nan] * 4, [nan, 1, nan, 1], [inf, 0, inf, 5], [-inf, -inf, -3e38, -inf], [nan, inf, -inf, 2],
                  [3e38, -3e38, 3.1e38, 0], [0.0, -0.0, 0.0, -0.0]])
    for f in FILTERS + [(inf, 0, 1.0, 0.0), (nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0), (1e30, 0, 0.9, 0.0),
                        (1.0, 2, nan, nan), (1.0, 0xFFFFFFFF, 2.0, 7.0), (1.0, 0, -1.0, -1.0), (1e-42, 0, 0.9, 0.0)]:
        for u in (0.0, 0.3, 0.7, 1.0, nan, -1.0, 2.0):
            check_draw(be, tens, l, [f] * 8, [u] * 8)


def test_draw_depends_on_its_row_alone(be, tens):
    """The same rows alone, in a batch and in another order: the same tokens and bits."""
    rng = np.random.default_rng(8)
    l = (rng.standard_normal((40, 65536)) * 2).astype(np.float32)
    f, u = [FILTERS[r % 5] for r in range(40)], rng.random(40).astype(np.float32)
    tok, logp = run_draw(be, tens, l, f, u)
    back = np.arange(39, -1, -1)
    t2, p2 = run_draw(be, tens, l[back], [f[r] for r in back], u[back])
    assert np.array_equal(tok, t2[back]) and np.array_equal(logp, p2[back])
    for r in (0, 13, 39):
        t1, p1 = run_draw(be, tens, l[r:r + 1], [f[r]], u[r:r + 1])
        assert t1[0] == tok[r] and p1[0] == logp[r]


def test_draw_without_logp_and_store_filter(be, tens):
    import rsv
    rng = np.random.default_rng(9)
    l = rng.standard_normal((3, 999)).astype(np.float32)
    f = tens(n=12)
    rows = [(0.5, 10, 0.9, 0.0), (1.5, 0, 1.0, 0.25), (0.0, 0, 1.0, 0.0)]
    for r, (t, k, p, m) in enumerate(rows):
        be.call("rsv_store_filter", f, r, t, k, p, m)
    u = np.array([0.2, 0.9, 0.4], np.float32)
    tok, work = tens(n=3, dtype=rsv.U32), tens(n=max(1, rsv.hip_lib().rsv_logits_work(999, 3)))
    be.call("rsv_sample_rand_batch", tens(l), tok, 999, f, tens(u), NONE, work, 3)
    want = [draw64(l[r], *[np.float32(v) if j != 1 else v for j, v in enumerate(rows[r])], u[r])[0] for r in range(3)]
    assert be.get(tok, 3, rsv.U32).tolist() == want
    with pytest.raises(rsv.RsvError, match="needs"):
        be.call("rsv_store_filter", f, 3, 1.0, 0, 1.0, 0.0)


def test_draw_refusals(be, tens):
    import rsv
    l, tok, f, u, p, w = tens(n=20), tens(n=2, dtype=rsv.U32), tens(n=8), tens(n=2), tens(n=2), tens(n=4096)
    ok = [l, tok, 10, f, u, p, w, 2]
    be.call("rsv_sample_rand_batch", *ok)
    for match, at, v in [("n=0", 2, 0), ("n=1048577", 2, 1048577), ("needs", 2, 11), ("0 rows", 7, 0), ("needs", 7, 3),
                         ("unknown tensor", 0, NONE), ("must be F32 or F16", 0, tok), ("unknown tensor", 1, NONE),
                         ("needs", 3, u), ("unknown tensor", 4, NONE), ("unknown tensor", 6, NONE),
                         ("another operand", 5, u), ("another operand", 1, u), ("another operand", 6, l)]:
        if match == "another operand" and at == 6:
            ok2 = list(ok)
            ok2[0] = ok2[6]
            with pytest.raises(rsv.RsvError, match=match):
                be.call("rsv_sample_rand_batch", *ok2)
            continue
        with pytest.raises(rsv.RsvError, match=match):
            be.call("rsv_sample_rand_batch", *[v if i == at else a for i, a in enumerate(ok)])


# ------------------------------------------------- log-probabilities
def logprobs64(l, tok):
    l = np.where(np.isnan(l), -np.inf, np.asarray(l, np.float64))
    n, m = l.size, l.max()
    if tok >= n:
        return 0.0, 0, 0.0
    rank = np.count_nonzero(l > l[tok]) + np.count_nonzero(l[:tok] == l[tok])
    if l[tok] == -np.inf:
        return -np.inf, rank, 0.0
    with np.errstate(invalid="ignore"):
        z = np.where(l == m, 0.0, l - m)
    e = np.exp(z)
    lp = z[tok] - math.log(e.sum())
    # roundings: z and its exp (an fp32 argument's rounding acts times its size) by each term's share of the sum, the
    # sum's own (at most n / 256 additions follow each other), the logarithm's and the result's
    far = float((e * np.abs(np.where(np.isfinite(z), z, 0))).sum() / e.sum())
    return lp, rank, U * (2 * abs(z[tok]) + 3 * far + n / 256 + 16 + 2 * abs(lp))


def run_logprobs(be, tens, l, tok, kind="f32", rank=True):
    import rsv
    rows, n = l.shape
    lp, rk = tens(n=rows), tens(n=rows, dtype=rsv.U32) if rank else NONE
    work = tens(n=max(1, rsv.hip_lib().rsv_logits_work(n, rows)))
    be.call("rsv_token_logprobs", tens.real(l, kind), tens.u32(tok), n, lp, rk, work, rows)
    return be.get(lp, rows), be.get(rk, rows, rsv.U32) if rank else None


def check_logprobs(be, tens, l, tok, kind="f32"):
    l = np.asarray(l, np.float32)
    if kind == "f16":
        l = l.astype(np.float16).astype(np.float32)
    lp, rk = run_logprobs(be, tens, l, tok, kind)
    for r in range(len(l)):
        want, rank, off = logprobs64(l[r], int(tok[r]))
        assert rk[r] == rank, (r, rk[r], rank)
        # -6e38 is -inf in fp32 (its largest number is 3.4e38)
        assert lp[r] == np.float32(want) or abs(lp[r] - want) <= off, (r, lp[r], want, off)


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (2, 7), (5, 63), (4, 65), (9, 1000), (3, 4097), (7, 65529), (1, 65536),
                                    (40, 65536), (2, 131072), (1, 1048576), (600, 1024), (1500, 33)])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_logprobs(be, tens, rows, n, kind):
    rng = np.random.default_rng(rows + n)
    l = rng.standard_normal((rows, n)) * rng.choice([0.0, 1.0, 5.0], (rows, 1))
    l[rng.random((rows, n)) < 0.05] = -np.inf
    if n > 4:
        l[1::3] = np.round(l[1::3])
    tok = rng.integers(0, n, rows).astype(np.uint32)
    l[np.arange(rows)[:-1:2], tok[:-1:2]] = 9.0
    tok[rows // 2::7] = NONE
    if rows > 3:
        tok[3] = n
    check_logprobs(be, tens, l, tok, kind)


def test_logprobs_non_finite_and_far(be, tens):
    inf, nan = np.inf, np.nan
    l = np.array([[-inf] * 5, [nan] * 5, [nan, 1, 2, nan, 1], [inf, 0, inf, 5, -inf], [3e38, -3e38, 0, 3e38, 1],
                  [-3e38, -3e38, -inf, nan, -3e38], [0.0, -0.0, 0.0, 0.0, -0.0], [100, 0, -100, 88, 3]])
    for t in range(5):
        check_logprobs(be, tens, l, np.full(8, t, np.uint32))
    lp, _ = run_logprobs(be, tens, l.astype(np.float32), np.full(8, 2, np.uint32), rank=False)
    lp2, _ = run_logprobs(be, tens, l.astype(np.float32), np.full(8, 2, np.uint32))
    assert np.array_equal(lp, lp2)


@pytest.mark.parametrize("entry", ["draw", "logprobs"])
def test_rows_past_32_bits(be, tens, entry):
    """Rows that start past 2^31 elements: the last rows of a tensor of 2^31 and more halves, the others not asked for
    (log-probabilities) or all alike (draws)."""
    import rsv
    torch = pytest.importorskip("torch")
    n, rows = 65536, 32772
    big = tens(n=n * rows, dtype=rsv.F16)  # zeros
    rng = np.random.default_rng(4)
    l = (rng.standard_normal((2, n)) * 2).astype(np.float16)
    p = ctypes.c_void_p()
    be.call("rsv_tensor_ptr", big, ctypes.byref(p))
    mem = type("M", (), {"__cuda_array_interface__": dict(shape=(2 * n,), typestr="<f2", version=2, strides=None,
                                                          data=(p.value + 2 * n * (rows - 2), False))})()
    torch.as_tensor(mem, device="cuda").copy_(torch.from_numpy(l.reshape(-1)))
    torch.cuda.synchronize()
    work = tens(n=max(1, rsv.hip_lib().rsv_logits_work(n, rows)))
    lp, whole = tens(n=rows), tens(n=rows, dtype=rsv.U32)
    if entry == "draw":
        f = np.tile(filters_of([(1.0, 0, 0.9, 0.0)]), (rows, 1))
        f[:-2, 0] = 0.0  # greedy
        u = np.full(rows, 0.37, np.float32)
        be.call("rsv_sample_rand_batch", big, whole, n, tens(f), tens(u), lp, work, rows)
        tok, got = be.get(whole, rows, rsv.U32), be.get(lp, rows)
        assert (tok[:-2] == 0).all() and (got[:-2] == 0).all()
        for r in (0, 1):
            want, p64 = draw64(l[r].astype(np.float32), np.float32(1), 0, np.float32(0.9), np.float32(0), u[0])
            assert tok[rows - 2 + r] == want and abs(got[rows - 2 + r] - p64) <= 2 * U * abs(p64) + 1e-9
        return
    tok = np.full(rows, NONE, np.uint32)
    tok[-2:] = [5, 60000]
    be.call("rsv_token_logprobs", big, tens.u32(tok), n, lp, whole, work, rows)
    got, rk = be.get(lp, rows), be.get(whole, rows, rsv.U32)
    assert (got[:-2] == 0).all() and (rk[:-2] == 0).all()
    for r in (0, 1):
        want, rank, off = logprobs64(l[r].astype(np.float32), int(tok[rows - 2 + r]))
        assert rk[rows - 2 + r] == rank and abs(got[rows - 2 + r] - want) <= off


def test_logprobs_refusals(be, tens):
    import rsv
    l, tok, p, r, w = tens(n=20), tens(n=2, dtype=rsv.U32), tens(n=2), tens(n=2, dtype=rsv.U32), tens(n=4096)
    ok = [l, tok, 10, p, r, w, 2]
    be.call("rsv_token_logprobs", *ok)
    for match, at, v in [("n=0", 2, 0), ("n=1048577", 2, 1048577), ("needs", 2, 11), ("0 rows", 6, 0), ("needs", 6, 3),
                         ("unknown tensor", 0, NONE), ("must be F32 or F16", 0, tok), ("unknown tensor", 1, NONE),
                         ("unknown tensor", 3, NONE), ("unknown tensor", 5, NONE), ("another operand", 4, tok),
                         ("another operand", 3, w)]:
        with pytest.raises(rsv.RsvError, match=match):
            be.call("rsv_token_logprobs", *[v if i == at else a for i, a in enumerate(ok)])


# ------------------------------------------------------- a served step
def test_served_step_eager_and_replayed(be, tens):
    """Head projection, adapters on it, a draw per row, its log-probability under the whole row and the embedding of
    the token for the next step: eager and captured, each replay with other requests, settings and random numbers."""
    import rsv
    rng = np.random.default_rng(17)
    B, C, V, na, rank = 12, 256, 1600, 5, 16
    W = np.asarray(rng.standard_normal((V, C)) * C ** -0.5, np.float16).astype(np.float32)
    emb = np.asarray(rng.standard_normal((V, C)), np.float16).astype(np.float32)
    w, e = tens.f16(W), tens.f16(emb)
    c = Adapters(tens, rng, B, na, rank, [(C, V)], "f16", "f32", inplace=True)
    c.host[0][0] *= 2
    c.upload()
    x, logits = c.jobs[0].x, c.jobs[0].y
    f, u, tok = tens(n=4 * B), tens(n=B), tens(n=B, dtype=rsv.U32)
    logp, full, rank_t, nxt = tens(n=B), tens(n=B), tens(n=B, dtype=rsv.U32), tens(n=B * C)
    work = tens(n=max(1, rsv.hip_lib().rsv_logits_work(V, B)))

    def step():
        be.call("rsv_gemm_ex", x, w, None, logits, B, V, C, 0, NONE, NONE, NONE)
        c.call(be)
        be.call("rsv_sample_rand_batch", logits, tok, V, f, u, logp, work, B)
        be.call("rsv_token_logprobs", logits, tok, V, full, rank_t, work, B)
        be.call("rsv_gather_rows_device_f16", e, nxt, tok, C, B)

    def put(t, a, u32=False):
        a = np.ascontiguousarray(a, np.uint32 if u32 else np.float32)
        be.call("rsv_upload_u32" if u32 else "rsv_upload", t,
                a.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32 if u32 else ctypes.c_float)), a.size)

    def set_inputs():
        c.ids = rng.integers(0, na + 1, B).astype(np.uint32)
        X = np.asarray(rng.standard_normal((B, C)), np.float16).astype(np.float32)
        c.host[0][2] = X
        s = dict(f=[FILTERS[i] for i in rng.integers(0, 10, B)], u=rng.random(B).astype(np.float32))
        put(c.t_ids, c.ids, True)
        put(x, X)
        put(f, filters_of(s["f"]))
        put(u, s["u"])
        return s

    def read():
        return [be.get(logits, B * V), be.get(tok, B, rsv.U32), be.get(logp, B), be.get(full, B),
                be.get(rank_t, B, rsv.U32), be.get(nxt, B * C)]

    def check(s, got):
        lg, tk, lp, fl, rk, nx = got
        lg = lg.reshape(B, V)
        c.host[0][3] = np.zeros((B, V), np.float32)
        z, off = c.want()[0]
        X = c.host[0][2].astype(np.float64)
        z = z + X @ W.astype(np.float64).T
        off = off + (C + 2) * U * (np.abs(X) @ np.abs(W).astype(np.float64).T + np.abs(z))
        assert (np.abs(lg - z) <= off).all()
        for r in range(B):
            row = [np.float32(v) if j != 1 else v for j, v in enumerate(s["f"][r])]
            want, p = draw64(lg[r], *row, s["u"][r])
            assert tk[r] == want and abs(lp[r] - p) <= 2 * U * abs(p) + 1e-9
            p64, rank64, o = logprobs64(lg[r], want)
            assert rk[r] == rank64 and abs(fl[r] - p64) <= o
            assert np.array_equal(nx[r * C:(r + 1) * C], emb[want])

    s = set_inputs()
    step()
    check(s, read())
    be.call("rsv_graph_begin")
    step()
    be.call("rsv_graph_end")
    for _ in range(3):
        s = set_inputs()
        be.call("rsv_graph_replay")
        got = read()
        check(s, got)
        step()
        for a, b in zip(got, read()):
            assert np.array_equal(a, b)


def test_two_lanes_at_once(be, tens):
    """The three operators on both lanes in turn, each lane with its own work area and outputs: the results of one lane
    alone."""
    import rsv
    rng = np.random.default_rng(23)
    n, rows = 65529, 9
    c = [Adapters(tens, np.random.default_rng(s), 130, 5, 16, [(520, 264)], "f16", "f32") for s in (1, 2)]
    l = rng.standard_normal((rows, n)).astype(np.float32) * 3
    f, u, logits = [FILTERS[i % 10] for i in range(rows)], rng.random(rows), tens(l)
    t_f, t_u = tens(filters_of(f)), tens(u)
    out = [(tens(n=rows, dtype=rsv.U32), tens(n=rows), tens(n=rows), tens(n=rsv.hip_lib().rsv_logits_work(n, rows)))
           for _ in range(2)]
    for a in c:
        a.upload()
    be.call("rsv_synchronize")
    try:
        for rep in range(4):
            for lane in (0, 1):
                be.call("rsv_lane_select", lane)
                tok, logp, full, work = out[lane]
                c[lane].call(be)
                be.call("rsv_sample_rand_batch", logits, tok, n, t_f, t_u, logp, work, rows)
                be.call("rsv_token_logprobs", logits, tok, n, full, NONE, work, rows)
        for lane in (0, 1):
            be.call("rsv_lane_select", lane)
            be.call("rsv_synchronize")
    finally:
        be.call("rsv_lane_select", 0)
    for lane in (0, 1):
        c[lane].check(be)
    a, b = [[be.get(o[0], rows, rsv.U32), be.get(o[1], rows), be.get(o[2], rows)] for o in out]
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    for r in range(rows):
        want, lp = draw64(l[r], *[np.float32(v) if j != 1 else v for j, v in enumerate(f[r])], np.float32(u[r]))
        assert a[0][r] == want and abs(a[1][r] - lp) <= 2 * U * abs(lp) + 1e-9
