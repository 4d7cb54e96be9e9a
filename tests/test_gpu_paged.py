"""The paged cache on the GPU (append, attention, accept), through the C ABI, against its definitions in 64 bits
(paged_reference.py). What moves without arithmetic has to be equal; the rest is held to bounds derived from the
roundings."""
import numpy as np
import pytest

import paged_reference as R
from yalama_b200 import engine as E

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
D = 128
F = E.StepFault
EPS16 = 2.0 ** -11  # half a step of FP16


def stream():
    return torch.cuda.current_stream().cuda_stream


def half(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float16)).cuda()


def ints(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def garbage(*shape):
    """FP16 that no sum survives: NaN, infinities of both signs, in a pattern."""
    x = np.full(shape, np.nan, np.float16)
    x.reshape(-1)[1::3] = np.inf
    x.reshape(-1)[2::3] = -np.inf
    return x


class Device:
    """Device side of a step: the pools (all garbage but for what `k`, `v` put there) and the step's arrays."""

    def __init__(self, step, hkv, layers=None, max_rows=None, rows=None, fault=True):
        self.step, self.hkv = step, hkv
        shape = (step.n_pages, hkv, step.page, D) if layers is None else (layers, step.n_pages, hkv, step.page, D)
        self.host = {x: garbage(*shape) for x in "kv"}
        self.row_start, self.length, self.table = ints(step.start), ints(step.lengths), ints(step.table)
        self.parent = None if step.trees is None else ints(step.flat_parents())
        self.fault = torch.zeros(1, dtype=torch.int32, device="cuda") if fault else None
        self.max_rows = max(step.rows + [0]) if max_rows is None else max_rows
        self.rows = step.total if rows is None else rows
        self.pool = None

    def put(self, kind, s, j, x):
        """Slots j of request s: x [len(j), hkv, 128]."""
        page, place = self.step.place(s, j)
        self.host[kind][..., page, :, place, :] = x

    def upload(self):
        self.pool = {x: half(self.host[x]) for x in "kv"}
        self.cache = E.paged_cache(ptr(self.pool["k"]), ptr(self.pool["v"]), self.step.n_pages, self.step.page, self.hkv)
        self.handle()
        return self

    def handle(self):
        self.st = E.paged_step(ptr(self.row_start), ptr(self.length), ptr(self.table), ptr(self.parent),
                               len(self.step.rows), self.table.shape[1], self.rows, self.max_rows, ptr(self.fault))

    def faults(self):
        return F(int(self.fault.item()))


def append(d, q, k, v, hq, norms=(None, None), rope=(None, None), out=None, eps=1e-6, s=None):
    if out is None:
        out = torch.full((d.rows, hq, D), 7.0, dtype=torch.float16, device="cuda")
    E.check(E.lib().ylm_k_paged_append(d.cache, d.st, ptr(q), q.stride(0) if q is not None else 0, ptr(k), k.stride(0),
                                       ptr(v), v.stride(0), hq, ptr(norms[0]), ptr(norms[1]), eps, ptr(rope[0]),
                                       ptr(rope[1]), 0 if rope[0] is None else rope[0].shape[0], ptr(out),
                                       out.stride(0), stream() if s is None else s), "append")
    return out


def workspace(d, hq):
    return torch.empty(E.paged_attention_workspace(d.cache, d.st, hq), dtype=torch.uint8, device="cuda")


def attend(d, q, hq, out=None, ws="own", s=None):
    if out is None:
        out = torch.full((d.rows, hq, D), 7.0, dtype=torch.float16, device="cuda")
    w = workspace(d, hq) if isinstance(ws, str) else ws
    E.check(E.lib().ylm_k_paged_attention(d.cache, d.st, ptr(q), q.stride(0), hq, ptr(out), out.stride(0), ptr(w),
                                          0 if w is None else w.numel(), stream() if s is None else s), "attention")
    return out


def accept(d, tokens, picks, layers, stride=0, s=None):
    n = len(d.step.rows)
    o = {"accepted": torch.full((n, d.max_rows), -9, dtype=torch.int32, device="cuda"),
         "n": torch.full((n,), -9, dtype=torch.int32, device="cuda"),
         "next": torch.full((n,), -9, dtype=torch.int64, device="cuda"),
         "length": torch.full((n,), -9, dtype=torch.int32, device="cuda")}
    E.check(E.lib().ylm_k_paged_accept(d.cache, d.st, ptr(tokens), ptr(picks), layers, stride, ptr(o["accepted"]),
                                       ptr(o["n"]), ptr(o["next"]), ptr(o["length"]), stream() if s is None else s),
            "accept")
    return o


def rope_tables(rng, max_pos):
    a = np.arange(max_pos)[:, None] * 500000.0 ** (-np.arange(64) / 64)
    return np.cos(a).astype(np.float16), np.sin(a).astype(np.float16)


# ---------------------------------------------------------------- append

APPENDS = [  # page, lengths, rows, trees, hq, hkv, norm, rope, pad
    (16, [0], [1], None, 4, 2, False, True, 0),
    (16, [15], [1], None, 1, 1, True, True, 0),
    (16, [16, 0, 31], [1, 1, 1], None, 8, 4, False, True, 2),
    (32, [5, 40], [70, 1], None, 14, 2, True, True, 0),
    (64, [3, 100, 63, 0], [7, 0, 30, 128], "random", 16, 8, True, True, 5),
    (128, [1000, 127], [128, 2], "line", 9, 3, False, True, 1),
    (16, [33, 7, 90], [20, 33, 64], "forest", 32, 8, False, True, 0),
    (16, [2, 9], [9, 5], "star", 5, 5, True, False, 0),
    (32, [11], [300], None, 2, 1, False, False, 4),
    (64, list(range(70)), [1] * 70, None, 2, 1, True, True, 3),
    (16, [i % 37 for i in range(1100)], [i % 3 for i in range(1100)], None, 1, 1, False, True, 0),
]


def make(rng, page, lengths, rows, trees, pad=0, **kw):
    t = None if trees is None else [R.tree(rng, trees, x) for x in rows]
    return R.Step(rng, page, lengths, rows, t, pad, **kw)


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"page{c[0]}-{c[4]}-{c[5]}-{c[3]}")
def test_append(case):
    page, lengths, rows, trees, hq, hkv, norm, rope, pad = case
    rng = np.random.default_rng(page + len(lengths))
    st = make(rng, page, lengths, rows, trees, pad)
    d = Device(st, hkv).upload()
    x = (rng.standard_normal((st.total, hq + 2 * hkv, D)) * np.exp2(rng.uniform(-3, 3, (st.total, 1, 1)))).astype(np.float16)
    x[::5, :, 3] *= 50
    w = [(1 + 0.3 * rng.standard_normal(D)).astype(np.float16) if norm else None for _ in "qk"]
    tab = rope_tables(rng, max(n + t for n, t in zip(lengths, rows)) + 1) if rope else (None, None)
    dx = half(x)
    before = {k: d.pool[k].clone() for k in "kv"}
    out = append(d, dx[:, :hq], dx[:, hq:hq + hkv], dx[:, hq + hkv:], hq, [None if a is None else half(a) for a in w],
                 [None if a is None else half(a) for a in tab])
    want_k, want_v = before["k"].cpu().numpy().astype(np.float64), before["v"].cpu().numpy()
    tol_k = np.zeros_like(want_k)
    want_q = np.full((st.total, hq, D), 7.0)
    tol_q = np.zeros_like(want_q)
    for s in range(len(rows)):
        at = slice(int(st.start[s]), int(st.start[s + 1]))
        y = np.concatenate([R.norm(x[at, :hq], w[0], 1e-6), R.norm(x[at, hq:hq + hkv], w[1], 1e-6)], 1)
        mag = abs(y)
        if rope:
            y, mag = R.rotate(y, lengths[s] + st.depths(s), *tab)
        # FP32: the norm's sum of 128 squares and its rsqrt (2 steps) stay below 2^-21.5, two products and a sum below
        # 2^-22.4: 2^-20 of the magnitudes together. Then one rounding to FP16 (2^-25: half its smallest step).
        tol = EPS16 * abs(y) + (2.0 ** -20 * mag if norm or rope else 0) + 2.0 ** -25
        want_q[at], tol_q[at] = y[:, :hq], tol[:, :hq]
        p, c = st.place(s, lengths[s] + np.arange(rows[s]))
        want_k[p, :, c], tol_k[p, :, c] = y[:, hq:], tol[:, hq:]
        want_v[p, :, c] = x[at, hq + hkv:]
    got = out.cpu().numpy().astype(np.float64)
    assert np.all(abs(got - want_q) <= tol_q)
    np.testing.assert_array_equal(d.pool["v"].cpu().numpy().view(np.uint16), want_v.view(np.uint16))
    got = d.pool["k"].cpu().numpy().astype(np.float64)
    new = tol_k > 0
    assert np.all(abs(got[new] - want_k[new]) <= tol_k[new])
    np.testing.assert_array_equal(got[~new], want_k[~new])
    assert d.faults() == 0


def test_append_in_place_and_keys_alone():
    rng = np.random.default_rng(0)
    st = make(rng, 16, [5, 20], [3, 4], None)
    tab = [half(a) for a in rope_tables(rng, 64)]
    x = half(rng.standard_normal((7, 8, D)))
    a, b = Device(st, 2).upload(), Device(st, 2).upload()
    want = append(a, x[:, :4], x[:, 4:6], x[:, 6:], 4, rope=tab)
    append(b, None, x[:, 4:6], x[:, 6:], 0, rope=tab)
    for k in "kv":
        assert torch.equal(a.pool[k].view(torch.int16), b.pool[k].view(torch.int16))
    append(b, x[:, :4], x[:, 4:6], x[:, 6:], 4, rope=tab, out=x[:, :4])
    assert torch.equal(x[:, :4], want)


def bad_step():
    """Seven requests, of which the second to fifth cannot be served, and one has a page that is not in the pool."""
    rng = np.random.default_rng(5)
    st = R.Step(rng, 16, [5, 30, 7, 0, 9, 40, 3], [3, 2, 2, 4, 2, 10, 2])
    return st


def break_step(d):
    st = d.step
    length = np.array(st.lengths)
    length[1], length[2], length[4] = -4, 16 * d.table.shape[1] - 1, 2 ** 31 - 1
    d.length.copy_(ints(length))
    d.max_rows = 10
    d.table[5, 2] = d.step.n_pages  # slots 32..47 of request 5
    d.table[0, 1:] = -2 ** 31
    d.handle()


def test_append_leaves_out_what_cannot_be_served():
    st = bad_step()
    good, d = Device(st, 1).upload(), Device(st, 1).upload()
    rng = np.random.default_rng(1)
    x = half(rng.standard_normal((st.total, 3, D)))
    want = append(good, x[:, :1], x[:, 1:2], x[:, 2:], 1)
    break_step(d)
    out = append(d, x[:, :1], x[:, 1:2], x[:, 2:], 1)
    assert d.faults() == F.BAD_REQUEST | F.BAD_PAGE
    for s in range(7):
        at = slice(int(st.start[s]), int(st.start[s + 1]))
        assert torch.equal(out[at], want[at]) if s in (0, 3, 5, 6) else bool((out[at] == 7).all())
        for kind in "kv":
            for j in range(st.lengths[s], st.lengths[s] + st.rows[s]):
                p, c = st.place(s, j)
                a, b = good.pool[kind][p, :, c], d.pool[kind][p, :, c]
                if s in (0, 3, 6) or (s == 5 and j >= 48):
                    assert torch.equal(a, b)
                else:
                    assert not bool(torch.isfinite(b).any())


@pytest.mark.parametrize("starts", [[0, 3, 2, 9], [-1, 2, 4, 9], [0, 3, 4, 100], [0, 8, 8, 9], [5, 4, 3, 2],
                                    [2 ** 31 - 1, -2 ** 31, 0, 4]], ids=str)
def test_impossible_row_starts_are_left_out(starts):
    # rows that overlap, decrease or lie outside the buffers: whatever is served lies within them
    rng = np.random.default_rng(2)
    st = make(rng, 16, [5, 5, 5], [3, 3, 3], None)
    d = Device(st, 1, max_rows=5).upload()
    d.row_start.copy_(ints(starts))
    x = half(rng.standard_normal((9, 3, D)))
    append(d, x[:, :1], x[:, 1:2], x[:, 2:], 1)
    assert d.faults() == F.BAD_REQUEST
    d.fault.zero_()
    attend(d, x[:, :1], 1)
    assert d.faults() & F.BAD_REQUEST
    d.fault.zero_()
    o = accept(d, ints(np.zeros(9), np.int64), ints(np.ones(9), np.int64), 1)
    assert d.faults() & F.BAD_REQUEST
    served = [a >= 0 and a < b <= 9 and b - a <= 5 for a, b in zip(starts, starts[1:])]
    assert o["n"].cpu().tolist() == [int(x) for x in served]
    assert o["length"].cpu().tolist() == [5 + int(x) for x in served]


def test_append_bad_parents_and_positions():
    rng = np.random.default_rng(3)
    st = R.Step(rng, 16, [10, 30], [4, 4], [[-1, 0, 1, 2], [-1, 0, 0, 1]])
    tab = rope_tables(rng, 33)
    x = rng.standard_normal((8, 3, D)).astype(np.float16)
    good, d = Device(st, 1).upload(), Device(st, 1).upload()
    dx, dt = half(x), [half(a) for a in tab]
    want = append(good, dx[:, :1], dx[:, 1:2], dx[:, 2:], 1, rope=dt)
    # row 2 of request 0 names itself, row 3 a later one: both count as first rows, at position 10
    d.parent.copy_(ints([-1, 0, 2, 7, -1, 0, 0, 1]))
    out = append(d, dx[:, :1], dx[:, 1:2], dx[:, 2:], 1, rope=dt)
    assert d.faults() == F.BAD_PARENT
    y, _ = R.rotate(x[2:4, :1].astype(np.float64), np.array([10, 10]), *tab)
    assert np.all(abs(out[2:4].cpu().numpy() - y) <= EPS16 * abs(y) + 2.0 ** -18)
    keep = [0, 1, 4, 5, 6, 7]
    assert torch.equal(out[keep], want[keep])
    # positions 30..32 exist, 33 does not
    d = Device(R.Step(rng, 16, [10, 31], [4, 4], st.trees), 1).upload()
    out = append(d, dx[:, :1], dx[:, 1:2], dx[:, 2:], 1, rope=dt)
    assert d.faults() == F.BAD_POSITION
    assert bool((out[7] == 7).all()) and not bool((out[:7] == 7).any())


# ---------------------------------------------------------------- attention


def bounds(out, pv, mag, v, see):
    """Scores: 128-term FP32 sums, each of the 8 steps of the matrix unit off by at most 2^-23 of the sum of magnitudes
    twice over: 2^-19 of the largest slot's magnitudes, which covers the scaling and the difference from the reference
    score, too; exp2 below 2^-20. A weight is then off by twice that (numerator and sum). The sums over n slots: 2^-24
    of the magnitudes for each addition. Weights enter the product rounded to FP16: by 2^-11 of themselves, of those
    below 2^-25 of the row's largest by 2^-36 of that one. The result is rounded."""
    n = v.shape[0]
    dp = 2 * (2.0 ** -19 * mag + 2.0 ** -20) + 2 * n * 2.0 ** -24
    small = 2.0 ** -36 * np.stack([abs(v[see[i]]).sum(0) if see[i].any() else np.zeros(D) for i in range(see.shape[0])])
    return EPS16 * abs(out) + (EPS16 + dp)[..., None] * pv + small[:, None] + 2.0 ** -24


def fill(rng, d, scale=1.0):
    """Random keys (a few strong channels) and values in all slots of the step, new ones included."""
    vals = []
    for s, (n, t) in enumerate(zip(d.step.lengths, d.step.rows)):
        k = rng.standard_normal((n + t, d.hkv, D)) * scale
        k[:, :, 5] *= 4
        v = rng.standard_normal((n + t, d.hkv, D)) * np.exp2(rng.uniform(-4, 4, (n + t, 1, 1)))
        k, v = k.astype(np.float16), v.astype(np.float16)
        d.put("k", s, np.arange(n + t), k)
        d.put("v", s, np.arange(n + t), v)
        vals.append((k, v))
    d.upload()
    return vals


def check(d, vals, q, out, hidden=None, requests=None):
    """out [rows, hq, 128] against the definition; rows of no request as they were."""
    st = d.step
    hq = q.shape[1]
    G = hq // d.hkv
    got = out.float().cpu().numpy().astype(np.float64)
    touched = np.zeros(got.shape[0], bool)
    for s in range(len(st.rows)) if requests is None else requests:
        at = slice(int(st.start[s]), int(st.start[s + 1]))
        touched[at] = True
        if st.rows[s] == 0:
            continue
        see = st.sees(s)
        if hidden is not None:
            see = see & ~hidden[s]
        for g in range(d.hkv):
            k, v = (x[:, g].astype(np.float64) for x in vals[s])
            want, pv, mag = R.attention(q[at, g * G:(g + 1) * G].astype(np.float64), k, v, see)
            err = abs(got[at, g * G:(g + 1) * G] - want)
            tol = bounds(want, pv, mag, v, see)
            assert np.all(err <= tol), (s, g, float(np.nanmax(err / tol)), np.argwhere(~(err <= tol))[:4].tolist())
    assert np.all(got[~touched] == 7)


ATTENDS = [  # page, lengths, rows, trees, hq, hkv, pad
    (16, [0], [1], None, 1, 1, 0),
    (16, [1], [1], None, 8, 8, 0),
    (16, [15, 16, 17], [1, 1, 1], None, 4, 2, 2),
    (16, [126, 127, 128, 129], [1, 1, 1, 1], None, 6, 2, 0),
    (128, [127, 128, 0, 255], [1, 0, 1, 1], None, 32, 8, 3),
    (32, [300, 2000, 5], [1, 1, 1], None, 28, 4, 0),
    (64, [3500], [1], None, 5, 1, 0),
    (16, list(range(0, 650, 13)), [1] * 50, None, 7, 1, 1),
    (16, [0], [2], "star", 4, 4, 0),
    (64, [200, 63], [64, 9], "random", 4, 2, 0),
    (16, [120, 1, 700], [17, 128, 40], "random", 16, 4, 2),
    (32, [100], [128], "line", 3, 1, 0),
    (128, [1000], [33], "forest", 32, 8, 0),
    (64, [0, 60, 500], [64, 64, 64], "forest", 14, 2, 1),
    (32, [10, 40], [31, 5], "random", 40, 1, 0),
    (16, [70], [3], "star", 128, 1, 0),
    (16, [0], [300], None, 4, 1, 0),
    (64, [129, 0], [257, 130], None, 6, 2, 0),
    (128, [511, 2], [200, 129], None, 10, 5, 1),
    (16, [90], [1], None, 127, 1, 0),
    (32, [77, 6], [5, 90], None, 100, 1, 0),
    (16, [1500, 3, 40, 800, 0, 9], [1, 64, 0, 1, 30, 2], None, 8, 2, 4),
    (64, [4000, 100], [1, 300], None, 8, 2, 0),
    (16, [i % 50 for i in range(1000)], [i % 2 for i in range(1000)], None, 2, 1, 0),
    # many units and items for every CTA: short and long requests side by side
    (16, [(i * 977) % 4001 for i in range(60)], [1] * 60, None, 14, 7, 2),
    (64, [(i * 613) % 2500 for i in range(24)], [(i * 7) % 60 + 1 for i in range(24)], "random", 16, 4, 0),
    (32, [(i * 613) % 2500 for i in range(24)], [(i * 5) % 27 + 1 for i in range(24)], "forest", 16, 4, 1),
    (128, [40000, 3], [1, 2], None, 6, 2, 0),
    (32, [700, 0, 2500], [400, 150, 333], None, 8, 2, 0),
    (16, [30 * i for i in range(130)], [1 + i % 2 for i in range(130)], None, 4, 2, 0),
]


@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: f"page{c[0]}-{c[4]}-{c[5]}-{c[3]}")
def test_attention(case):
    page, lengths, rows, trees, hq, hkv, pad = case
    rng = np.random.default_rng(page + hq)
    d = Device(make(rng, page, lengths, rows, trees, pad), hkv)
    vals = fill(rng, d)
    q = rng.standard_normal((d.rows, hq, D)).astype(np.float16)
    dq = half(q)
    out = attend(d, dq, hq)
    check(d, vals, q, out)
    assert d.faults() == 0
    # the same bits again, without a workspace of the caller's, and in a step whose bounds are wider than its rows
    assert torch.equal(attend(d, dq, hq, ws=None), out)
    if trees is None:
        d.max_rows += 37
        d.handle()
        check(d, vals, q, attend(d, dq, hq))


@pytest.mark.parametrize("scale", [0.0, 0.02, 30.0, 400.0])
def test_attention_from_flat_to_one_hot(scale):
    rng = np.random.default_rng(7)
    d = Device(make(rng, 16, [300, 40], [20, 40], "random"), 2)
    vals = fill(rng, d, scale)
    q = rng.standard_normal((d.rows, 8, D)).astype(np.float16)
    check(d, vals, q, attend(d, half(q), 8))


def test_attention_rising_scores():
    # every slot's score is above the one before: the softmax's reference has to follow all the way
    rng = np.random.default_rng(8)
    d = Device(make(rng, 32, [700], [40], None), 1)
    for rise in (0.01, 0.5, 3.0):
        vals = []
        k = np.zeros((740, 1, D))
        k[:, 0, 0] = np.arange(740) * rise
        v = rng.standard_normal((740, 1, D))
        vals.append((k.astype(np.float16), v.astype(np.float16)))
        for x, y in zip("kv", vals[0]):
            d.put(x, 0, np.arange(740), y)
        d.upload()
        q = np.zeros((40, 4, D), np.float16)
        q[:, :, 0] = [[11.3, -11.3, 1.0, 0.0]]
        check(d, vals, q, attend(d, half(q), 4))


def test_small_weights_far_below_the_largest_count():
    # one slot of weight 1 - 2^-9 whose values are 0, and thousands that share the rest
    n = 6000
    rng = np.random.default_rng(9)
    d = Device(make(rng, 64, [n - 1], [1], None), 1)
    k, v = np.zeros((n, 1, D), np.float16), rng.uniform(0.5, 1.5, (n, 1, D)).astype(np.float16)
    k[100, 0, 0] = 1
    v[100] = 0
    d.put("k", 0, np.arange(n), k)
    d.put("v", 0, np.arange(n), v)
    d.upload()
    q = np.zeros((1, 1, D), np.float16)
    q[0, 0, 0] = np.log(n * 512) * np.sqrt(D)
    check(d, [(k, v)], q, attend(d, half(q), 1))


@pytest.mark.parametrize("hq,hkv", [(2, 1), (32, 8)])
def test_what_hidden_slots_hold_does_not_matter(hq, hkv):
    # siblings that are NaN or infinite: rows that do not see them are as if they were not there, the others get them
    rng = np.random.default_rng(10)
    trees = [[-1, 0, 0, 1, 2, 3, 4, 0, -1] + [1] * 60]
    d = Device(R.Step(rng, 16, [100], [69], trees), hkv)
    vals = fill(rng, d)
    k, v = vals[0][0].copy(), vals[0][1].copy()
    k[100 + 2], v[100 + 1, :, 7], v[100 + 7, :, 9], v[100 + 8, :, ::2] = np.nan, np.inf, -np.inf, np.nan
    v[100 + 5, :, 7], v[100 + 68, :, 100:] = -np.inf, np.inf
    for x, y in zip("kv", (k, v)):
        d.put(x, 0, np.arange(169), y)
    d.upload()
    q = rng.standard_normal((69, hq, D)).astype(np.float16)
    out = attend(d, half(q), hq).float().cpu().numpy()
    with np.errstate(all="ignore"):
        for i in range(69):
            see = d.step.sees(0)[i:i + 1]
            for g in range(hkv):
                G = hq // hkv
                kk, vv = k[:, g].astype(np.float64), v[:, g].astype(np.float64)
                want, _, _ = R.attention(q[i:i + 1, g * G:(g + 1) * G].astype(np.float64), kk, vv, see)
                got = out[i, g * G:(g + 1) * G]
                np.testing.assert_array_equal(np.isnan(got), np.isnan(want[0]))
                np.testing.assert_array_equal(np.isposinf(got), np.isposinf(want[0]))
                np.testing.assert_array_equal(np.isneginf(got), np.isneginf(want[0]))
                fin = np.isfinite(want[0])
                clean = np.where(np.isfinite(vv), vv, 0)
                seen = see & np.isfinite(kk).all(1)
                w2, pv, mag = R.attention(q[i:i + 1, g * G:(g + 1) * G].astype(np.float64), np.nan_to_num(kk), clean, seen)
                tol = bounds(w2, pv, mag, clean, seen)[0]
                assert np.all(abs(got[fin] - want[0][fin]) <= tol[fin])


def test_infinities_and_nan_among_the_cached_tokens():
    rng = np.random.default_rng(11)
    d = Device(make(rng, 16, [200, 200, 200], [2, 2, 2], None), 1)
    vals = fill(rng, d)
    k, v = [x[0].copy() for x in vals], [x[1].copy() for x in vals]
    v[0][50, 0, 3], v[0][51, 0, 4], v[0][60, 0, 4] = np.inf, np.inf, -np.inf
    k[1][30, 0, 8] = np.nan
    k[2][30, 0, 8] = -np.inf  # a score of -inf where q is positive there (no weight), +inf (no softmax) elsewhere
    for s in range(3):
        d.put("k", s, np.arange(202), k[s])
        d.put("v", s, np.arange(202), v[s])
    d.upload()
    q = rng.standard_normal((6, 2, D)).astype(np.float16)
    q[4:, :, 8] = [[1, -1], [2, 0.5]]
    out = attend(d, half(q), 2).float().cpu().numpy()
    assert np.all(np.isposinf(out[:2, :, 3])) and np.all(np.isnan(out[:2, :, 4]))
    rest = np.ones(D, bool)
    rest[3:5] = False
    assert np.all(np.isfinite(out[:2][:, :, rest]))
    assert np.all(np.isnan(out[2:4]))
    assert np.all(np.isnan(out[4, 1])) and np.all(np.isfinite(out[[4, 5, 5], [0, 0, 1]]))
    hidden = np.zeros((2, 202), bool)
    hidden[:, 30] = True
    see = d.step.sees(2) & ~hidden
    kk = np.nan_to_num(k[2][:, 0].astype(np.float64), neginf=0)
    for i, h in ((0, 0), (1, 0), (1, 1)):
        want, pv, mag = R.attention(q[4 + i:5 + i, h:h + 1].astype(np.float64), kk, v[2][:, 0].astype(np.float64), see[i:i + 1])
        tol = bounds(want, pv, mag, v[2][:, 0].astype(np.float64), see[i:i + 1])
        assert np.all(abs(out[4 + i, h] - want[0, 0]) <= tol[0, 0])


def test_attention_pages_that_are_not_in_the_pool():
    rng = np.random.default_rng(12)
    for page, trees in ((16, None), (128, None), (32, "random")):
        d = Device(make(rng, page, [400, 300, 5, 700], [3, 20, 2, 130] if trees is None else [3, 20, 2, 100], trees), 2)
        vals = fill(rng, d)
        bad = [(0, 2), (0, 0), (1, 1), (2, 0), (3, 4), (3, 5)]
        for i, (s, p) in enumerate(bad):
            d.table[s, p] = (-1, d.step.n_pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
        hidden = []
        for s in range(4):
            h = np.zeros(d.step.lengths[s] + d.step.rows[s], bool)
            for x, p in bad:
                if x == s:
                    h[p * page:(p + 1) * page] = True
            hidden.append(h)
        q = rng.standard_normal((d.rows, 6, D)).astype(np.float16)
        out = attend(d, half(q), 6)
        check(d, vals, q, out, hidden)
        assert d.faults() == F.BAD_PAGE
        assert bool((out[23:25] == 0).all())  # request 2 has no other page


def test_attention_leaves_out_what_cannot_be_served():
    st = bad_step()
    d = Device(st, 1)
    rng = np.random.default_rng(13)
    vals = fill(rng, d)
    q = rng.standard_normal((d.rows, 2, D)).astype(np.float16)
    break_step(d)
    d.table[5, 2] = ints(st.table)[5, 2]
    check(d, vals, q, attend(d, half(q), 2), requests=[0, 3, 5, 6])
    assert d.faults() == F.BAD_REQUEST


def test_attention_strides_and_columns():
    rng = np.random.default_rng(14)
    d = Device(make(rng, 16, [77, 20], [5, 40], "random"), 2)
    vals = fill(rng, d)
    wide = half(rng.standard_normal((d.rows, 11, D)))
    out = torch.full((d.rows, 13, D), 7.0, dtype=torch.float16, device="cuda")
    attend(d, wide[:, 2:8], 6, out=out[:, 4:10])
    check(d, vals, wide[:, 2:8].cpu().numpy(), out[:, 4:10])
    assert bool((out[:, :4] == 7).all()) and bool((out[:, 10:] == 7).all())


def test_workspace_too_small_is_refused():
    d = Device(make(np.random.default_rng(0), 16, [500], [3], None), 1)
    fill(np.random.default_rng(0), d)
    need = E.paged_attention_workspace(d.cache, d.st, 4)
    if need == 0:
        pytest.skip("no workspace")
    q = half(np.zeros((3, 4, D)))
    with pytest.raises(E.YlmError, match="needed"):
        attend(d, q, 4, ws=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))


# ---------------------------------------------------------------- accept


@pytest.mark.parametrize("page,lengths,rows,trees,hkv,layers,pad", [
    (16, [0], [1], "random", 1, 1, 0), (16, [0], [8], "line", 2, 3, 0), (16, [15, 14, 30], [5, 0, 33], "random", 3, 2, 4),
    (64, [60, 100, 0, 3], [128, 20, 64, 1], "random", 2, 5, 0), (32, [31] * 9, [9] * 9, "forest", 1, 2, 1),
    (128, [120, 5], [128, 128], "line", 1, 1, 0), (16, [7, 40], [30, 12], "star", 8, 28, 0),
    (16, [i % 20 for i in range(700)], [i % 7 for i in range(700)], "random", 1, 2, 0),
    (16, [5, 9, 0], [300, 1, 0], None, 2, 2, 3), (32, [40], [64], "random", 2, 0, 0)], ids=lambda x: str(x)[:20])
@pytest.mark.parametrize("vocab", [2, 40])
def test_accept(page, lengths, rows, trees, hkv, layers, pad, vocab):
    rng = np.random.default_rng(page + sum(rows) + vocab)
    st = make(rng, page, lengths, rows, trees, pad)
    d = Device(st, hkv, max(layers, 1) + 1)  # a layer too many: it stays as it was
    shape = d.host["k"].shape
    bits = {x: rng.integers(0, 65536, shape).astype(np.uint16) for x in "kv"}
    d.host = {x: bits[x].view(np.float16) for x in "kv"}
    d.upload()
    # tokens of a small vocabulary: several children match, and long paths are accepted; ids beyond 32 bits, too
    tokens = rng.integers(0, vocab, st.total) + (1 << 40)
    picks = rng.integers(0, vocab, st.total) + (1 << 40)
    for s in range(len(rows)):
        for i, p in enumerate(st.parents(s)):
            if p >= 0 and rng.random() < 0.5:
                picks[st.start[s] + p] = tokens[st.start[s] + i]
    o = accept(d, ints(tokens, np.int64), ints(picks, np.int64), layers, int(np.prod(shape[1:])))
    for s in range(len(rows)):
        a = int(st.start[s])
        t = slice(a, a + rows[s])
        path = R.accept(st.parents(s), tokens[t], picks[t]) if rows[s] else []
        assert o["accepted"][s].cpu().tolist() == path + [-1] * (d.max_rows - len(path))
        assert int(o["n"][s]) == len(path) and int(o["length"][s]) == lengths[s] + len(path)
        assert int(o["next"][s]) == (picks[a + path[-1]] if path else -1)
        for j, i in enumerate(path):
            (pa, ca), (pb, cb) = st.place(s, lengths[s] + i), st.place(s, lengths[s] + j)
            for x in bits.values():
                x[:layers, pb, :, cb] = x[:layers, pa, :, ca]
    for x in "kv":
        np.testing.assert_array_equal(d.pool[x].cpu().numpy().view(np.uint16), bits[x])
    assert d.faults() == 0


def test_accept_leaves_out_what_cannot_be_served():
    rng = np.random.default_rng(15)
    trees = [[-1, 0, 0, 2, 3], [-1, 0, 0, 2, 3], [-1, 0, 5, -3, 0], [-1, 0, 0, 2, 3]]
    st = R.Step(rng, 16, [13, 14, 15, 20], [5] * 4, trees)
    d = Device(st, 1)
    vals = fill(rng, d)
    before = {x: d.pool[x].clone() for x in "kv"}
    length = np.array(st.lengths)
    length[0] = -1
    d.length.copy_(ints(length))
    d.table[1, 1] = d.step.n_pages + 5  # slots 16..31: of path 0, 2, 3, 4 only the first token's places are there
    tokens = np.tile([9, 1, 2, 3, 4], 4)
    picks = np.tile([2, 0, 3, 4, 77], 4)
    o = accept(d, ints(tokens, np.int64), ints(picks, np.int64), 1)
    assert d.faults() == F.BAD_REQUEST | F.BAD_PAGE | F.BAD_PARENT
    assert o["n"].cpu().tolist() == [0, 4, 1, 4]  # request 2's rows 2 and 3 follow nothing
    assert o["next"].cpu().tolist() == [-1, 77, 2, 77] and o["length"].cpu().tolist() == [-1, 18, 16, 24]
    for x, y in zip("kv", vals[3]):
        p, c = st.place(3, 20 + np.arange(4))
        want = y[20 + np.array([0, 2, 3, 4])]
        np.testing.assert_array_equal(d.pool[x][p, :, c].cpu().numpy(), want)
        for s in (0, 1, 2):
            p, _ = st.place(s, np.arange(0, st.lengths[s] + 5, 16))
            assert torch.equal(d.pool[x][p].view(torch.int16), before[x][p].view(torch.int16))


# ---------------------------------------------------------------- together


def test_drafted_tokens_over_several_steps():
    """Trees are appended, attended, accepted, step by step; the accepted tokens' outputs and cache are those of a second
    pool that gets them one by one."""
    rng = np.random.default_rng(16)
    hq, hkv, layers, page, steps, vocab = 8, 2, 3, 16, 6, 50
    tab = [half(a) for a in rope_tables(rng, 400)]
    embed = rng.standard_normal((vocab, hq + 2 * hkv, D)).astype(np.float16)  # a token's q, k, v before rotation
    lengths = [40, 5, 0]
    table = np.arange(3 * 20).reshape(3, 20)[:, ::-1].copy()

    class Pool:
        def __init__(self):
            self.k, self.v = (torch.zeros(layers, 60, hkv, page, D, dtype=torch.float16, device="cuda") for _ in "kv")
            self.caches = [E.paged_cache(ptr(self.k[i]), ptr(self.v[i]), 60, page, hkv) for i in range(layers)]

    a, b = Pool(), Pool()
    dtab = ints(table)

    def run(pool, length, tokens, parents):
        """One step of rows [request][row]; outputs of the last layer."""
        starts = np.concatenate([[0], np.cumsum([len(t) for t in tokens])])
        rows = int(starts[-1])
        keep = [ints(starts), ints(length), ints(np.concatenate(parents)) if parents is not None else None]
        st = E.paged_step(ptr(keep[0]), ptr(keep[1]), ptr(dtab), ptr(keep[2]), 3, 20, rows, max(len(t) for t in tokens))
        x = half(embed[np.concatenate(tokens)])
        out = torch.zeros(rows, hq, D, dtype=torch.float16, device="cuda")
        for i in range(layers):
            q = torch.empty(rows, hq, D, dtype=torch.float16, device="cuda")
            E.check(E.lib().ylm_k_paged_append(pool.caches[i], st, ptr(x), x.stride(0), ptr(x[:, hq:]), x.stride(0),
                                               ptr(x[:, hq + hkv:]), x.stride(0), hq, None, None, 0.0, ptr(tab[0]),
                                               ptr(tab[1]), 400, ptr(q), q.stride(0), stream()), "append")
            E.check(E.lib().ylm_k_paged_attention(pool.caches[i], st, ptr(q), q.stride(0), hq, ptr(out), out.stride(0),
                                                  None, 0, stream()), "attention")
        return st, keep, out, starts

    prompt = [rng.integers(0, vocab, n) for n in lengths]
    for pool in (a, b):
        run(pool, [0, 0, 0], [p if len(p) else np.zeros(0, np.int64) for p in prompt], None)
    last = [int(rng.integers(0, vocab)) for _ in range(3)]
    for step in range(steps):
        trees = [R.tree(rng, "random", int(rng.integers(3, 30))) for _ in range(3)]
        tokens = [np.concatenate([[last[s]], rng.integers(0, vocab, len(trees[s]) - 1)]) for s in range(3)]
        st, keep, out, starts = run(a, lengths, tokens, [np.array(t) for t in trees])
        # the model's picks, from logits whose largest is a child's token more often than not
        logits = torch.randn(int(starts[-1]), vocab, device="cuda").half()
        for s in range(3):
            for i, p in enumerate(trees[s]):
                if p >= 0 and rng.random() < 0.6:
                    logits[int(starts[s]) + p, int(tokens[s][i])] = 30
        picks = torch.empty(int(starts[-1]), 1, dtype=torch.int64, device="cuda")
        lp = torch.empty(int(starts[-1]), 1, device="cuda")
        E.check(E.lib().ylm_k_logprobs(ptr(logits), vocab, int(starts[-1]), vocab, None, None, 1, None, None, ptr(picks),
                                       ptr(lp), stream()), "logprobs")
        m = max(len(t) for t in tokens)
        res = [torch.empty(3, m, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda"),
               torch.empty(3, dtype=torch.int64, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")]
        flat = ints(np.concatenate(tokens), np.int64)
        E.check(E.lib().ylm_k_paged_accept(a.caches[0], st, ptr(flat), ptr(picks), layers, a.k.stride(0),
                                           *[ptr(x) for x in res], stream()), "accept")
        accepted, count = res[0].cpu().numpy(), res[1].cpu().numpy()
        for s in range(3):
            assert accepted[s, :count[s]].tolist() == R.accept(trees[s], tokens[s],
                                                               picks[int(starts[s]):int(starts[s + 1]), 0].cpu().numpy())
        # one by one in the other pool: a step for each depth, requests that are done have no row
        for j in range(int(count.max())):
            one = [tokens[s][[accepted[s, j]]] if j < count[s] else np.zeros(0, np.int64) for s in range(3)]
            at = [lengths[s] + min(j, int(count[s])) for s in range(3)]
            _, _, single, ss = run(b, at, one, None)
            for s in range(3):
                if j < count[s]:
                    x, y = single[int(ss[s])].float(), out[int(starts[s]) + int(accepted[s, j])].float()
                    # each is within 2^-11 |o| + 2^-11 sum p |v| of the same value: |v| stays below 6, plus dp
                    assert float((x - y).abs().max()) <= 4 * EPS16 * 6
        lengths = res[3].cpu().tolist()
        last = res[2].cpu().tolist()
        for s in range(3):
            j = torch.arange(lengths[s], device="cuda")
            p, c = dtab[s][j // page].long(), j % page
            for x, y in ((a.k, b.k), (a.v, b.v)):
                assert torch.equal(x[:, p, :, c], y[:, p, :, c])


def test_one_graph_serves_steps_of_other_lengths_and_trees():
    rng = np.random.default_rng(17)
    hq, hkv, page, seqs, rows = 8, 2, 16, 4, 60
    st = R.Step(rng, page, [200, 3, 90, 0], [20, 1, 9, 30], [R.tree(rng, "random", t) for t in (20, 1, 9, 30)])
    d = Device(st, hkv, max_rows=40, rows=rows)
    d.parent = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    d.upload()
    tab = [half(a) for a in rope_tables(rng, 700)]
    x = torch.zeros(rows, hq + 2 * hkv, D, dtype=torch.float16, device="cuda")
    q = torch.full((rows, hq, D), 7.0, dtype=torch.float16, device="cuda")
    out = torch.full((rows, hq, D), 7.0, dtype=torch.float16, device="cuda")
    # a pool and a table that hold every step
    big = 200
    d.pool = {k: half(garbage(big, hkv, page, D)) for k in "kv"}
    d.cache = E.paged_cache(ptr(d.pool["k"]), ptr(d.pool["v"]), big, page, hkv)
    d.table = torch.full((seqs, 48), -1, dtype=torch.int32, device="cuda")
    d.handle()
    ws = workspace(d, hq)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        append(d, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], hq, rope=tab, out=q)
        attend(d, q, hq, out=out, ws=ws)
    for lengths, t in (([200, 3, 90, 0], [20, 1, 9, 30]), ([0, 600, 1, 17], [1, 40, 0, 12]), ([5, 5, 5, 5], [0, 0, 0, 0]),
                       ([700 - 41, 0, 30, 2], [40, 1, 1, 1])):
        st = R.Step(rng, page, lengths, t, [R.tree(rng, "random", m) for m in t], pad=rows - sum(t))
        d.step = st
        assert st.n_pages <= big and st.table.shape[1] <= 48
        d.row_start.copy_(ints(st.start))
        d.length.copy_(ints(lengths))
        d.parent.copy_(ints(st.flat_parents()))
        d.table[:, :st.table.shape[1]] = ints(st.table)
        host = {k: garbage(big, hkv, page, D) for k in "kv"}
        cached = []
        for s, n in enumerate(lengths):
            kv = [rng.standard_normal((n, hkv, D)).astype(np.float16) for _ in "kv"]
            p, c = st.place(s, np.arange(n))
            for k, y in zip("kv", kv):
                host[k][p, :, c] = y
            cached.append(kv)
        for k in "kv":
            d.pool[k].copy_(half(host[k]))
        new = rng.standard_normal((rows, hq + 2 * hkv, D)).astype(np.float16)
        x.copy_(half(new))
        q.fill_(7.0)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        vals = []
        for s, n in enumerate(lengths):
            p, c = st.place(s, np.arange(n + t[s]))
            vals.append([d.pool[k].cpu().numpy()[p, :, c] for k in "kv"])
            np.testing.assert_array_equal(vals[s][1][n:], new[st.start[s]:st.start[s + 1], hq + hkv:])
        check(d, vals, q.cpu().numpy(), out)
        assert d.faults() == 0


def test_graphs_with_a_workspace_each_and_an_eager_call_between():
    rng = np.random.default_rng(21)
    made = []
    for i in range(2):
        st = make(rng, 16, [900, 33, 200], [20, 60, 7], "random")
        d = Device(st, 2)
        vals = fill(rng, d)
        q = rng.standard_normal((d.rows, 8, D)).astype(np.float16)
        tokens, picks = ints(rng.integers(0, 3, d.rows), np.int64), ints(rng.integers(0, 3, d.rows), np.int64)
        m = dict(d=d, vals=vals, q=q, dq=half(q), ws=workspace(d, 8), out=torch.full((d.rows, 8, D), 7.0, dtype=torch.float16, device="cuda"),
                 tokens=tokens, picks=picks, graph=torch.cuda.CUDAGraph())
        attend(d, m["dq"], 8, out=m["out"], ws=m["ws"])
        torch.cuda.synchronize()
        with torch.cuda.graph(m["graph"]):
            attend(d, m["dq"], 8, out=m["out"], ws=m["ws"])
            m["res"] = accept(d, tokens, picks, 0)
        made.append(m)
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for m, side in zip(made, sides):
            m["out"].record_stream(side)
            with torch.cuda.stream(side):
                m["graph"].replay()
        x = attend(made[0]["d"], made[0]["dq"], 8)  # meanwhile, on the current stream
    torch.cuda.synchronize()
    for m in made:
        check(m["d"], m["vals"], m["q"], m["out"])
        st = m["d"].step
        for s in range(3):
            a, b = int(st.start[s]), int(st.start[s + 1])
            path = R.accept(st.parents(s), m["tokens"][a:b].cpu().numpy(), m["picks"][a:b].cpu().numpy())
            assert m["res"]["accepted"][s, :len(path)].cpu().tolist() == path
    check(made[0]["d"], made[0]["vals"], made[0]["q"], x)


def test_a_workspace_for_max_rows_serves_steps_of_more_rows():
    rng = np.random.default_rng(22)
    d = Device(make(rng, 16, [300] * 12, [40] * 12, None), 2)
    fill(rng, d)
    big = E.paged_attention_workspace(d.cache, d.st, 8)
    d.rows = 40
    d.handle()
    assert E.paged_attention_workspace(d.cache, d.st, 8) == big


def test_two_streams_with_a_workspace_each():
    rng = np.random.default_rng(18)
    made = []
    for i in range(2):
        d = Device(make(rng, 32, [3000, 50, 900], [30, 4, 64], "random"), 2)
        vals = fill(rng, d)
        q = rng.standard_normal((d.rows, 8, D)).astype(np.float16)
        made.append((d, vals, q, half(q), workspace(d, 8), torch.cuda.Stream(), torch.full((d.rows, 8, D), 7.0, dtype=torch.float16, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for d, _, _, dq, ws, side, out in made:
            attend(d, dq, 8, out=out, ws=ws, s=side.cuda_stream)
    torch.cuda.synchronize()
    for d, vals, q, _, _, _, out in made:
        check(d, vals, q, out)


def test_offsets_beyond_32_bits():
    # 3 GB of pages: the last ones lie behind 2^31 bytes and 2^30 halves
    page, hkv, n_pages = 64, 4, 48000
    pool = {k: torch.empty(n_pages, hkv, page, D, dtype=torch.float16, device="cuda") for k in "kv"}
    rng = np.random.default_rng(19)
    st = R.Step(rng, page, [100, 40], [20, 9], [R.tree(rng, "random", t) for t in (20, 9)])
    st.table = np.where(st.table >= 0, n_pages - 1 - st.table, -1)
    st.n_pages = n_pages
    d = Device.__new__(Device)
    d.step, d.hkv, d.pool, d.rows, d.max_rows = st, hkv, pool, st.total, 20
    d.row_start, d.length, d.table, d.parent = ints(st.start), ints(st.lengths), ints(st.table), ints(st.flat_parents())
    d.fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    d.cache = E.paged_cache(ptr(pool["k"]), ptr(pool["v"]), n_pages, page, hkv)
    d.handle()
    vals = []
    for s, n in enumerate(st.lengths):
        p, c = st.place(s, np.arange(n + st.rows[s]))
        kv = [rng.standard_normal((n + st.rows[s], hkv, D)).astype(np.float16) for _ in "kv"]
        for k, y in zip("kv", kv):
            pool[k][torch.from_numpy(p).cuda(), :, torch.from_numpy(c).cuda()] = half(y)
        vals.append(kv)
    x = half(np.concatenate([np.stack([v[n:] for v in kv], 1) for kv, n in zip(vals, st.lengths)]))
    for k in "kv":  # the new rows by the operator
        pool[k][torch.from_numpy(st.place(0, 100 + np.arange(20))[0]).cuda(), :, torch.from_numpy(st.place(0, 100 + np.arange(20))[1]).cuda()] = 0
    append(d, None, x[:, 0], x[:, 1], 0)
    q = rng.standard_normal((st.total, 8, D)).astype(np.float16)
    check(d, vals, q, attend(d, half(q), 8))
    tokens = np.zeros(st.total)
    o = accept(d, ints(tokens, np.int64), ints(tokens, np.int64), 1)
    for s in range(2):
        path = R.accept(st.parents(s), np.zeros(st.rows[s]), np.zeros(st.rows[s]))
        assert o["accepted"][s, :len(path)].cpu().tolist() == path
        n = st.lengths[s]
        p, c = st.place(s, n + np.arange(len(path)))
        for k, y in zip("kv", vals[s]):
            got = pool[k][torch.from_numpy(p).cuda(), :, torch.from_numpy(c).cuda()].cpu().numpy()
            np.testing.assert_array_equal(got, y[n + np.array(path)])


def dominated(rng, seqs, units, hq, low=0.0):
    """Requests of one row over `units` units of 128 slots, keys of one channel, values of many sizes; enough of them that
    a CTA has several units of an item, and borders lie inside of others."""
    d = Device(make(rng, 16, [128 * units - 1] * seqs, [1] * seqs, None), 1)
    k = np.full((seqs, 128 * units, D), 0.0)
    k[:, :, 0] = low
    v = rng.standard_normal((seqs, 128 * units, D)).astype(np.float16)
    q = np.zeros((seqs, hq, D), np.float16)
    return d, k, v, q


def put_all(d, k, v):
    vals = []
    for s in range(len(d.step.rows)):
        x = [a[s][:, None].astype(np.float16) for a in (k, v)]
        for kind, y in zip("kv", x):
            d.put(kind, s, np.arange(y.shape[0]), y)
        vals.append(x)
    d.upload()
    return vals


def test_infinities_and_nan_under_a_dominating_score():
    # wherever the slot lies, a value that is not finite is not lost when another slot's score is 141 above its own
    rng = np.random.default_rng(23)
    cases = [(a, b, x) for a in range(4) for b in range(4) for x in (np.inf, -np.inf, np.nan)] * 6
    d, k, v, q = dominated(rng, len(cases), 4, 2)
    q[:, 0, 0] = 16
    for s, (a, b, x) in enumerate(cases):
        k[s, a * 128 + 5, 0] = 100
        v[s, b * 128 + 77, 3] = x
    vals = put_all(d, k, v)
    out = attend(d, half(q), 2)
    got = out.float().cpu().numpy()
    special = np.array([x for _, _, x in cases], np.float32)
    np.testing.assert_array_equal(got[:, 1, 3], special)  # every slot weighs the same
    assert not np.any(np.isfinite(got[:, 0, 3]))
    assert np.all(np.isnan(got[np.isnan(special), 0, 3]))
    # the other elements as if it were not there
    for x in vals:
        x[1][~np.isfinite(x[1])] = 0
    out[:, :, 3] = 0
    for s, x in enumerate(vals):
        x[1][:, :, 3] = 0
    check(d, vals, q, out)


@pytest.mark.parametrize("seqs", [1, 300])
def test_scores_that_are_nan_in_one_part_of_an_item(seqs):
    # rows that see one slot of the last unit, its score NaN, or -inf with a value that is NaN: the request in one CTA's
    # share, or every unit in another one's
    rng = np.random.default_rng(24)
    t = 20
    d = Device(R.Step(rng, 16, [256] * seqs, [t] * seqs, [[-1] * t] * seqs), 1)
    vals = fill(rng, d)
    q = rng.standard_normal((d.rows, 2, D)).astype(np.float16)
    q[:, :, 8] = 1
    for s in range(seqs):
        k, v = vals[s]
        k[256 + 3, 0, 20] = np.nan
        k[256 + 5, 0, 8] = -np.inf
        v[256 + 5, 0, 7] = np.nan
        d.put("k", s, np.arange(256 + t), k)
        d.put("v", s, np.arange(256 + t), v)
    d.upload()
    out = attend(d, half(q), 2)
    got = out.float().cpu().numpy().reshape(seqs, t, 2, D)
    assert np.all(np.isnan(got[:, 3])) and np.all(np.isnan(got[:, 5, :, 7]))
    # the rest as if those slots were hidden
    hidden = []
    for s in range(seqs):
        k, v = vals[s]
        k[~np.isfinite(k)], v[~np.isfinite(v)] = 0, 0
        h = np.zeros(256 + t, bool)
        h[[256 + 3, 256 + 5]] = True
        hidden.append(h)
    clean = out.clone().view(seqs, t, 2, D)
    clean[:, 3] = 0
    clean[:, 5, :, 7] = 0
    for s in range(seqs):
        for g, h in ((i, j) for i in range(t) for j in range(2)):
            see = d.step.sees(s)[g:g + 1] & ~hidden[s]
            kk, vv = vals[s][0][:, 0].astype(np.float64), vals[s][1][:, 0].astype(np.float64)
            want, pv, mag = R.attention(q[s * t + g:s * t + g + 1, h:h + 1].astype(np.float64), kk, vv, see)
            ok = np.ones(D, bool)
            ok[7] = g != 5
            if g != 3:
                err = abs(got[s, g, h] - want[0, 0])[ok]
                assert np.all(err <= bounds(want, pv, mag, vv, see)[0, 0][ok])


def test_scores_whose_steps_are_as_far_apart_as_weights_reach():
    # scores of 2^29 + 64 j (before the scale): neighbours in FP32, with weights 2^8 apart
    rng = np.random.default_rng(26)
    d, k, v, q = dominated(rng, 200, 6, 2)
    q[:, :, 0], q[:, :, 1] = 2.0 ** 14, [8, -8]
    k[:, :, 0], k[:, :, 1] = 2.0 ** 15, 8 * (np.arange(768) // 256)
    vals = put_all(d, k, v)
    out = attend(d, half(q), 2)
    # the large product is the same for every slot and both are powers of two: no score is rounded, and without
    # it the weights are the same
    small = [(x[0].copy(), x[1]) for x in vals]
    for x in small:
        x[0][:, :, 0] = 0
    check(d, small, q, out)


def test_values_at_the_ends_of_fp16():
    # one slot a unit counts, each stream's next one up to 2^4.8 times as much as its last: the reference stays behind,
    # weights are rounded, and what they weigh is the largest there is
    rng = np.random.default_rng(25)
    d, k, v, q = dominated(rng, 200, 6, 8, low=-200)
    k[:, 9::128, 0] = np.arange(6) // 2
    q[:, :, 0] = rng.uniform(0.5, 4.8, (200, 8)) * np.log(2) * np.sqrt(D)
    v[:, :, ::2], v[:, :, 1::2] = 65504, -65504
    vals = put_all(d, k, v)
    out = attend(d, half(q), 8)
    assert bool(torch.isfinite(out).all())
    check(d, vals, q, out)


@pytest.mark.parametrize("trees", [False, True])
def test_prompt_pieces_beside_single_tokens_and_trees(trees):
    """One step holds pieces of prompts, single tokens and drafted ones. The picks of given rows are set to the next given
    token, so that all of them are accepted; the cache then holds each request's tokens in order."""
    rng = np.random.default_rng(27)
    hq, hkv, page, layers, vocab, most = 4, 2, 16, 2, 40, 128 if trees else 300
    prompts = [rng.integers(0, vocab, n) for n in ((250, 1, 90, 128) if trees else (700, 1, 90, 300))]
    seqs, ld = 4, 60
    tab = [half(a) for a in rope_tables(rng, 900)]
    embed = rng.standard_normal((vocab, hq + 2 * hkv, D)).astype(np.float16)  # a token's q, k, v before rotation
    table = rng.permutation(seqs * ld).reshape(seqs, ld)
    dtab = ints(table)
    pools = [[torch.zeros(layers, seqs * ld, hkv, page, D, dtype=torch.float16, device="cuda") for _ in "kv"] for _ in range(2)]

    def run(pool, lengths, tokens, parents, max_rows):
        starts = np.concatenate([[0], np.cumsum([len(t) for t in tokens])])
        rows = int(starts[-1])
        keep = [ints(starts), ints(lengths), None if parents is None else ints(np.concatenate(parents))]
        st = E.paged_step(ptr(keep[0]), ptr(keep[1]), ptr(dtab), ptr(keep[2]), seqs, ld, rows, max_rows)
        x = half(embed[np.concatenate(tokens)])
        out = torch.zeros(rows, hq, D, dtype=torch.float16, device="cuda")
        q = torch.empty_like(out)
        for i in range(layers):
            c = E.paged_cache(ptr(pool[0][i]), ptr(pool[1][i]), seqs * ld, page, hkv)
            E.check(E.lib().ylm_k_paged_append(c, st, ptr(x), x.stride(0), ptr(x[:, hq:]), x.stride(0),
                                               ptr(x[:, hq + hkv:]), x.stride(0), hq, None, None, 0.0, ptr(tab[0]),
                                               ptr(tab[1]), 900, ptr(q), q.stride(0), stream()), "append")
            E.check(E.lib().ylm_k_paged_attention(c, st, ptr(q), q.stride(0), hq, ptr(out), out.stride(0), None, 0,
                                                  stream()), "attention")
        return st, keep, out, starts

    lengths, last, at = [0] * seqs, [0] * seqs, [0] * seqs
    history, given_outs = [[] for _ in range(seqs)], {}
    for step in range(12):
        tokens, parents, given = [], [], []
        for s, p in enumerate(prompts):
            left = p[at[s]:]
            if len(left):  # a piece of the prompt, as long as the step allows
                tokens.append(left[:int(rng.integers(1, most + 1))])
                parents.append(list(range(-1, len(tokens[-1]) - 1)))
            else:
                t = 1 if s == 1 else int(rng.integers(2, 30))
                tokens.append(np.concatenate([[last[s]], rng.integers(0, vocab, t - 1)]))
                parents.append(R.tree(rng, "random", t) if trees else list(range(-1, t - 1)))
            given.append(len(left) > 0)
        st, keep, out, starts = run(pools[0], lengths, tokens, parents if trees else None, most)
        rows = int(starts[-1])
        logits = torch.randn(rows, vocab, device="cuda").half()
        for s in range(seqs):
            for i, p in enumerate(parents[s]):
                if p >= 0 and rng.random() < 0.6:
                    logits[int(starts[s]) + p, int(tokens[s][i])] = 30
        picks = torch.empty(rows, dtype=torch.int64, device="cuda")
        lp = torch.empty(rows, device="cuda")
        E.check(E.lib().ylm_k_logprobs(ptr(logits), vocab, rows, vocab, None, None, 1, None, None, ptr(picks), ptr(lp),
                                       stream()), "logprobs")
        model = picks.cpu().numpy()
        flat = ints(np.concatenate(tokens), np.int64)
        for s in range(seqs):
            if given[s]:
                a, b = int(starts[s]), int(starts[s + 1])
                picks[a:b - 1] = flat[a + 1:b]
        res = [torch.empty(seqs, most, dtype=torch.int32, device="cuda"), torch.empty(seqs, dtype=torch.int32, device="cuda"),
               torch.empty(seqs, dtype=torch.int64, device="cuda"), torch.empty(seqs, dtype=torch.int32, device="cuda")]
        first = E.paged_cache(ptr(pools[0][0]), ptr(pools[0][1]), seqs * ld, page, hkv)
        E.check(E.lib().ylm_k_paged_accept(first, st, ptr(flat), ptr(picks), layers, pools[0][0].stride(0),
                                           *[ptr(x) for x in res], stream()), "accept")
        accepted, count, following, new = (x.cpu().numpy() for x in res)
        for s in range(seqs):
            a, t = int(starts[s]), len(tokens[s])
            path = list(range(t)) if given[s] else R.accept(parents[s], tokens[s], model[a:a + t])
            assert accepted[s].tolist() == path + [-1] * (most - len(path)) and count[s] == len(path)
            assert new[s] == lengths[s] + len(path) and following[s] == model[a + path[-1]]
            for i in path:
                given_outs[s, len(history[s])] = out[a + i].float()
                history[s].append(int(tokens[s][i]))
            if given[s]:
                at[s] += t
            last[s] = int(following[s])
        lengths = new.tolist()
    assert all(at[s] == len(prompts[s]) for s in range(seqs)) and min(lengths) > 1
    # every request's tokens as one chain
    _, _, out, starts = run(pools[1], [0] * seqs, [np.array(h) for h in history], None, max(lengths))
    for s in range(seqs):
        p, c = dtab[s][torch.arange(lengths[s], device="cuda") // page].long(), torch.arange(lengths[s], device="cuda") % page
        for x, y in zip(*pools):
            assert torch.equal(x[:, p, :, c], y[:, p, :, c])
        for j in range(lengths[s]):
            # each is within 2^-11 |o| + 2^-11 sum p |v| of the same value: |v| stays below 6, plus dp
            assert float((given_outs[s, j] - out[int(starts[s]) + j].float()).abs().max()) <= 4 * EPS16 * 6


@pytest.mark.parametrize("trees", [None, "random"])
def test_requests_that_share_the_pages_of_a_prefix(trees):
    # pages below the new rows' are of two requests and more, in a step that could have more rows: attention sees them
    # for each, and append and accept leave them as they are
    rng = np.random.default_rng(28)
    page, prefix, hkv, hq = 32, 256, 2, 8
    own, rows = [0, 40, 300, 7, 1000, 31], [1] * 6 if trees is None else [1, 20, 64, 9, 2, 33]
    st = make(rng, page, [prefix + n for n in own], rows, trees, 3)
    st.table[1:4, :prefix // page] = st.table[0, :prefix // page]
    st.table[5, :prefix // page] = st.table[4, :prefix // page]
    d = Device(st, hkv, max_rows=128)
    vals = []
    for s, n in enumerate(st.lengths):
        k, v = (rng.standard_normal((n + rows[s], hkv, D)).astype(np.float16) for _ in "kv")
        if s in (1, 2, 3, 5):
            k[:prefix], v[:prefix] = (x[:prefix] for x in vals[0 if s < 4 else 4])
        d.put("k", s, np.arange(n), k[:n])
        d.put("v", s, np.arange(n), v[:n])
        vals.append((k, v))
    d.upload()
    before = {x: d.pool[x].clone() for x in "kv"}
    new = [half(np.concatenate([x[i][n:] for x, n in zip(vals, st.lengths)] + [np.zeros((3, hkv, D))])) for i in range(2)]
    append(d, None, new[0], new[1], 0)
    q = rng.standard_normal((d.rows, hq, D)).astype(np.float16)
    check(d, vals, q, attend(d, half(q), hq))
    tokens = ints(np.zeros(d.rows), np.int64)
    accept(d, tokens, tokens, 1)  # every row's lowest child
    for s, n in enumerate(st.lengths):
        path = R.accept(st.parents(s), [0] * rows[s], [0] * rows[s])
        p, c = st.place(s, n + np.arange(len(path)))
        for x, y in zip("kv", vals[s]):
            np.testing.assert_array_equal(d.pool[x].cpu().numpy()[p, :, c], y[n + np.array(path)])
            common = st.table[s, :prefix // page]
            assert torch.equal(d.pool[x][common].view(torch.int16), before[x][common].view(torch.int16))
    assert d.faults() == 0
