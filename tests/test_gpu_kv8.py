"""The 8-bit K/V cache on the GPU (store, attention, eviction), through the C ABI, against its definitions in 64 bits
(kv8_reference.py). Codes and scales have to be equal: with power-of-two scales every step but one rounding is exact."""
import ctypes

import numpy as np
import pytest

import kv8_reference as R
from yalama_b200 import engine as E

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
D = 128
FMTS = ["e4m3", "int8"]


def stream():
    return torch.cuda.current_stream().cuda_stream


def half(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float16)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


class DeviceCache:
    """Device buffers of a cache; codes start as `fill` (NaN of E4M3, -1 of INT8) and scales as NaN, so that
    anything read that no store wrote shows."""

    def __init__(self, fmt, block, cap, hkv, fill=0xFF):
        self.fmt, self.block, self.cap, self.hkv = fmt, block, cap, hkv
        nb = -(-cap // block)
        self.code = {x: torch.full((hkv, cap, D), fill, dtype=torch.uint8, device="cuda") for x in "kv"}
        self.scale = {x: torch.full((hkv, nb), float("nan"), device="cuda") for x in "kv"}
        self.h = E.kv8_cache(ptr(self.code["k"]), ptr(self.code["v"]), ptr(self.scale["k"]), ptr(self.scale["v"]),
                             fmt, block, cap, hkv)

    def store(self, k, v, slot, s=None):
        E.check(E.lib().ylm_k_kv8_store(self.h, ptr(k), k.stride(0), ptr(v), v.stride(0), k.shape[0], slot,
                                        stream() if s is None else s), "store")

    def numbers(self, x):
        return R.numbers(self.code[x].cpu().numpy(), self.fmt)

    def same_as(self, ref, n):
        """Slots [0, n) and their scales equal the reference's; all behind untouched."""
        nb = -(-n // self.block)
        for x in "kv":
            np.testing.assert_array_equal(self.numbers(x)[:, :n], ref.num[x][:, :n])
            np.testing.assert_array_equal(self.scale[x].cpu().numpy()[:, :nb], ref.scale[x][:, :nb])
            assert bool((self.code[x][:, n:] == 0xFF).all())
            assert bool(torch.isnan(self.scale[x][:, nb:]).all())


def attend(c, q, t, n, mask=None, acc=None, out=None, ws="own", s=None):
    hq = q.shape[1]
    if out is None:
        out = torch.full((t, hq * D), float("nan"), dtype=torch.float16, device="cuda")
    need = E.kv8_attention_workspace(c.h, hq, t, n, acc is not None)
    w = torch.empty(need, dtype=torch.uint8, device="cuda") if ws == "own" else ws
    E.check(E.lib().ylm_k_kv8_attention(c.h, ptr(q), q.stride(0), hq, t, n, ptr(mask), ptr(acc), ptr(out),
                                        out.stride(0), ptr(w), 0 if w is None else w.numel(),
                                        stream() if s is None else s), "attention")
    return out


def evict(c, d, acc, acc_dst, n, keep, sink, recent, kept, s=None):
    E.check(E.lib().ylm_k_kv8_evict(c.h, d.h, ptr(acc), ptr(acc_dst), n, keep, sink, recent, ptr(kept),
                                    stream() if s is None else s), "evict")


def rows(rng, t, hkv, spread=1.0):
    """FP16 rows whose magnitude differs from token to token, with a few strong channels."""
    x = rng.standard_normal((t, hkv, D)) * np.exp2(rng.uniform(-3, 3, (t, 1, 1)) * spread)
    x[:, :, 5] *= 8
    return x.astype(np.float16)


def bits(hidden):
    w = np.zeros((hidden.size + 31) // 32, np.uint32)
    for i in np.nonzero(hidden)[0]:
        w[i >> 5] |= np.uint32(1) << np.uint32(i & 31)
    return torch.from_numpy(w.view(np.int32)).cuda()


def filled(rng, fmt, block, cap, hkv, n, spread=1.0):
    """A device cache and its reference with n random tokens."""
    c, ref = DeviceCache(fmt, block, cap, hkv), R.Cache(fmt, block, cap, hkv)
    k, v = rows(rng, n, hkv, spread), rows(rng, n, hkv, spread)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    return c, ref


# ---------------------------------------------------------------- store


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hkv,pieces", [(1, [1]), (2, [1, 1, 1]), (3, [15, 2, 33, 1, 127]), (8, [200, 129]),
                                        (2, [16, 16, 64, 128, 1])], ids=str)
def test_store(fmt, block, hkv, pieces):
    rng = np.random.default_rng(block * 100 + hkv)
    n = sum(pieces)
    c, ref = DeviceCache(fmt, block, n + 40, hkv), R.Cache(fmt, block, n + 40, hkv)
    slot = 0
    for t in pieces:
        k, v = rows(rng, t, hkv), rows(rng, t, hkv)
        c.store(half(k), half(v), slot)
        ref.store(k.astype(np.float64), v.astype(np.float64), slot)
        slot += t
    c.same_as(ref, n)


@pytest.mark.parametrize("fmt", FMTS)
def test_store_token_by_token_with_growing_magnitudes(fmt):
    # every token doubles the scale at least: the older ones are rescaled each time
    rng = np.random.default_rng(1)
    c, ref = DeviceCache(fmt, 16, 64, 2), R.Cache(fmt, 16, 64, 2)
    for i in range(20):
        k = (rng.standard_normal((1, 2, D)) * 2.0 ** (i % 16 - 8)).astype(np.float16)
        v = (rng.standard_normal((1, 2, D)) * 2.0 ** (4 - i % 16)).astype(np.float16)
        c.store(half(k), half(v), i)
        ref.store(k.astype(np.float64), v.astype(np.float64), i)
    c.same_as(ref, 20)


@pytest.mark.parametrize("fmt", FMTS)
def test_store_every_half_rounds_to_the_nearest_code(fmt):
    # all finite FP16 magnitudes against each power of two as the block's largest value
    every = np.arange(0, 0x7C00, dtype=np.uint16).view(np.float16)
    for top in (2.0 ** -24, 2.0 ** -14, 0.875, 1.0, 1.75, 1.984375, 1.9853515625, 448.0, 65504.0):
        x = every[every <= top]
        t = -(-x.size // D)
        k = np.zeros((t, 1, D), np.float16)
        k.reshape(-1)[:x.size] = x
        k[::16, 0, 0] = top  # the largest value of every block of 16
        c, ref = DeviceCache(fmt, 16, t, 1), R.Cache(fmt, 16, t, 1)
        c.store(half(k), half(-k), 0)
        ref.store(k.astype(np.float64), -k.astype(np.float64), 0)
        c.same_as(ref, t)


@pytest.mark.parametrize("fmt", FMTS)
def test_store_zeros_infinities_and_nan(fmt):
    k = np.zeros((40, 1, D), np.float16)
    k[20, 0, 3], k[21, 0, 4], k[22, 0, 5] = np.inf, -np.inf, np.nan
    v = np.zeros((40, 1, D), np.float16)
    v[17, 0, 7], v[18, 0, 7] = np.nan, 3
    c, ref = DeviceCache(fmt, 16, 64, 1), R.Cache(fmt, 16, 64, 1)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    c.same_as(ref, 40)
    assert float(c.scale["k"][0, 0]) == 0 and float(c.scale["k"][0, 2]) == 0
    # a token of ordinary size into the block of zeros
    k = rows(np.random.default_rng(0), 1, 1)
    c.store(half(k), half(k), 40)
    ref.store(k.astype(np.float64), k.astype(np.float64), 40)
    c.same_as(ref, 41)


def test_store_takes_columns_of_a_fused_projection_and_refills_a_block():
    rng = np.random.default_rng(3)
    qkv = (rng.standard_normal((70, 9, D))).astype(np.float16)
    d = half(qkv)
    c, ref = DeviceCache("e4m3", 32, 96, 2), R.Cache("e4m3", 32, 96, 2)
    c.store(d[:, 5:7], d[:, 7:9], 0)
    ref.store(qkv[:, 5:7].astype(np.float64), qkv[:, 7:9].astype(np.float64), 0)
    c.same_as(ref, 70)
    # a new sequence from slot 0: the old scales of a block that starts with it do not count
    small = (rows(rng, 32, 2) * np.float16(0.01)).astype(np.float16)
    c.store(half(small), half(small), 0)
    ref.store(small.astype(np.float64), small.astype(np.float64), 0)
    c.same_as(ref, 70)


# ---------------------------------------------------------------- attention

EPS16 = 2.0 ** -11  # half a step of FP16


def bounds(out, pv, mag, acc):
    """Scores: 128-term FP32 sums, each of the 8 steps of the matrix unit off by at most 2^-23 of the sum of magnitudes
    twice over (alignment and rounding): 2^-19 mag at most, and the same for exp2's argument and result, below 2^-20.
    A probability is then off by twice that (numerator and sum); P enters P V rounded to FP16; the result is rounded."""
    dp = 2 * (2.0 ** -19 * mag + 2.0 ** -20)
    tol_out = EPS16 * np.abs(out) + (EPS16 + dp)[..., None] * pv + 2.0 ** -24
    return tol_out, dp.max()


def check_attention(c, ref, q, t, n, hidden=None, acc=None, **kw):
    hid = np.zeros(n, bool) if hidden is None else hidden[:n]
    before = None if acc is None else acc.cpu().numpy().astype(np.float64)
    got = attend(c, half(q), t, n, None if hidden is None else bits(hidden), acc, **kw)
    out, w, pv, mag = R.attention(q.astype(np.float64), ref.values("k", n), ref.values("v", n), t, hid)
    tol, dp = bounds(out, pv, mag, acc)
    err = np.abs(got.float().cpu().numpy().astype(np.float64).reshape(out.shape) - out)
    assert np.all(err <= tol), float((err / tol).max())
    if acc is not None:
        after = acc.cpu().numpy().astype(np.float64)
        want = before.copy()
        want[:, :n] += w
        # the weights' own error, and one rounding for each of the additions into a slot
        lim = dp * w + (1 + q.shape[0] * q.shape[1] / c.hkv) * 2.0 ** -24 * np.abs(want[:, :n])
        err = np.abs(after[:, :n] - want[:, :n])
        assert np.all(err <= lim + 1e-30), float((err / (lim + 1e-30)).max())
        np.testing.assert_array_equal(after[:, n:], before[:, n:])
    return got


SHAPES = [  # hq, hkv, t, n, block
    (1, 1, 1, 1, 16), (8, 8, 1, 2, 16), (24, 8, 1, 15, 32), (16, 8, 1, 16, 16), (16, 8, 1, 17, 128), (4, 2, 1, 63, 64),
    (4, 2, 1, 64, 64), (4, 2, 1, 65, 64), (28, 4, 1, 129, 32), (64, 8, 1, 300, 128), (14, 2, 1, 1000, 16),
    (32, 8, 1, 2085, 64), (9, 1, 1, 77, 32), (12, 1, 1, 512, 16), (16, 1, 1, 200, 64), (17, 1, 1, 130, 16),
    (40, 1, 1, 95, 32), (128, 1, 1, 70, 16), (4, 2, 2, 2, 16), (4, 2, 7, 7, 16), (32, 8, 3, 40, 32),
    (28, 4, 5, 333, 64), (64, 8, 8, 515, 128), (8, 8, 16, 100, 16), (8, 1, 16, 129, 32), (14, 2, 13, 700, 64),
    (32, 8, 65, 190, 64), (6, 2, 200, 200, 32), (24, 8, 1, 1024, 32), (12, 1, 1, 1025, 16), (14, 2, 5, 2300, 64),
    (4, 2, 1, 897, 16), (16, 2, 2, 1000, 128), (33, 1, 4, 61, 16), (128, 1, 2, 64, 16), (2, 2, 129, 400, 128),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,t,n,block", SHAPES)
def test_attention(hq, hkv, t, n, block, fmt):
    rng = np.random.default_rng(hq * 1000 + n)
    c, ref = filled(rng, fmt, block, n + 37, hkv, n, 0.4)
    q = rng.standard_normal((t, hq, D)).astype(np.float16)
    plain = check_attention(c, ref, q, t, n)
    # the same with weights kept, and with hidden slots; the outputs do not depend on whether weights are kept
    acc = torch.rand(hkv, n + 37, device="cuda")
    again = check_attention(c, ref, q, t, n, None, acc)
    assert float((again.float() - plain.float()).abs().max()) <= 2 ** -10 * float(plain.float().abs().max())
    hidden = rng.random(n + 20) < 0.3
    check_attention(c, ref, q, t, n, hidden, acc)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,n", [(1, 70), (5, 130), (20, 20), (1, 1400), (3, 1100), (9, 1301)])
def test_attention_hidden_slots_may_hold_anything(fmt, t, n):
    rng = np.random.default_rng(n)
    c, ref = filled(rng, fmt, 16, n + 50, 2, n)
    q = rng.standard_normal((t, 8, D)).astype(np.float16)
    hidden = rng.random(n) < 0.5
    hidden[16:32] = True  # a whole block, whose scales are NaN too
    for x in "kv":
        c.code[x][:, torch.from_numpy(hidden).cuda().nonzero()[:, 0]] = 0x7F
        c.scale[x][:, 1] = float("nan")
    acc = torch.zeros(2, n + 50, device="cuda")
    check_attention(c, ref, q, t, n, hidden, acc)
    assert bool((acc[:, :n][:, torch.from_numpy(hidden).cuda()] == 0).all())


@pytest.mark.parametrize("t,n", [(1, 40), (6, 300), (40, 64), (1, 1200), (3, 1500), (12, 1100)])
def test_attention_rows_that_see_nothing_are_zero(t, n):
    rng = np.random.default_rng(n)
    c, ref = filled(rng, "e4m3", 32, n, 2, n)
    q = rng.standard_normal((t, 4, D)).astype(np.float16)
    acc = torch.rand(2, n, device="cuda")
    keep = acc.clone()
    out = attend(c, half(q), t, n, bits(np.ones(n, bool)), acc)
    assert bool((out == 0).all()) and torch.equal(acc, keep)
    # only the last slot open: the earlier tokens see nothing, the last one sees it alone
    hidden = np.ones(n, bool)
    hidden[-1] = False
    got = check_attention(c, ref, q, t, n, hidden, acc)
    if t > 1:
        assert bool((got[:-1] == 0).all())
    want = ref.values("v", n)[:, -1].repeat(2, 0).reshape(-1)
    np.testing.assert_allclose(got[-1].float().cpu().numpy(), want, rtol=2.0 ** -10, atol=1e-7)


@pytest.mark.parametrize("hq,t,n", [(2, 5, 100), (8, 3, 64), (8, 9, 33), (4, 40, 130), (2, 5, 1200), (8, 4, 1153)])
def test_attention_nan_of_a_later_token_stays_out_of_the_earlier_ones(hq, t, n):
    # NaN in a key makes every output of the tokens that see it NaN, NaN in a value that dimension of theirs
    rng = np.random.default_rng(n)
    hkv = 2
    k, v = rows(rng, n, hkv, 0.4), rows(rng, n, hkv, 0.4)
    v[n - 3, 0, 17] = v[n - 1, 1, 100] = v[n - 2, 1, 3] = np.nan
    k[n - 1, 0, 50] = np.nan
    c = DeviceCache("e4m3", 16, n + 20, hkv)
    c.store(half(k), half(v), 0)
    ref = R.Cache("e4m3", 16, n + 20, hkv)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    q = rng.standard_normal((t, hq, D)).astype(np.float16)
    kv, vv = ref.values("k", n), ref.values("v", n)
    out, _, pv, mag = R.attention(q.astype(np.float64), np.nan_to_num(kv), np.nan_to_num(vv), t, np.zeros(n, bool))
    bad = np.zeros((t, hq, D), bool)
    G = hq // hkv
    bad[t - 3:, :G, 17] = bad[t - 1:, G:, 100] = bad[t - 2:, G:, 3] = True
    bad[t - 1, :G] = True
    got = attend(c, half(q), t, n).float().cpu().numpy().reshape(out.shape)
    np.testing.assert_array_equal(np.isnan(got), bad)
    tol, _ = bounds(out, pv, mag, None)
    assert np.all((np.abs(got - out) <= tol)[~bad])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [400, 1300])
@pytest.mark.parametrize("sharp", [1.0, 30.0])
def test_attention_values_of_very_different_scales(fmt, sharp, n):
    # first tokens that take most of the weight with values near zero, and blocks of values 2^20 apart
    rng = np.random.default_rng(int(sharp))
    hkv, hq = 2, 8
    k = rng.standard_normal((n, hkv, D)).astype(np.float16)
    v = rng.standard_normal((n, hkv, D))
    v[:16] *= 2.0 ** -14
    v[16:32] *= 2.0 ** -10
    v[48:64] *= 2.0 ** 6
    v[64:80] = 0
    v = v.astype(np.float16)
    q = (rng.standard_normal((1, hq, D)) * 0.3).astype(np.float16)
    for h in range(hq):
        q[0, h] = q[0, h] + np.float16(0.02 * sharp) * k[3, h // 4]
    for lo, hi in ((0, n), (0, 48), (0, 90)):
        c, ref = DeviceCache(fmt, 16, n, hkv), R.Cache(fmt, 16, n, hkv)
        c.store(half(k[lo:hi]), half(v[lo:hi]), 0)
        ref.store(k[lo:hi].astype(np.float64), v[lo:hi].astype(np.float64), 0)
        check_attention(c, ref, q, 1, hi - lo, None, torch.zeros(hkv, n, device="cuda"))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [190, 1190])
def test_attention_of_large_scores(fmt, n):
    # scores in the thousands: one slot takes everything
    rng = np.random.default_rng(7)
    c, ref = filled(rng, fmt, 64, n + 10, 1, n)
    q = (rng.standard_normal((3, 4, D)) * 60).astype(np.float16)
    check_attention(c, ref, q, 3, n, None, torch.zeros(1, n + 10, device="cuda"))


@pytest.mark.parametrize("n", [280, 1280])
def test_attention_strided_rows_and_untouched_neighbours(n):
    rng = np.random.default_rng(11)
    c, ref = filled(rng, "int8", 32, n + 20, 4, n)
    qkv = rng.standard_normal((6, 20, D)).astype(np.float16)  # 12 query heads, then keys and values
    d = half(qkv)
    out = torch.full((6, 14 * D), 7.0, dtype=torch.float16, device="cuda")
    attend(c, d[:, :12], 6, n, out=out[:, :12 * D])
    want, _, pv, mag = R.attention(qkv[:, :12].astype(np.float64), ref.values("k", n), ref.values("v", n), 6,
                                   np.zeros(n, bool))
    tol, _ = bounds(want, pv, mag, None)
    assert np.all(np.abs(out[:, :12 * D].float().cpu().numpy().reshape(want.shape) - want) <= tol)
    assert bool((out[:, 12 * D:] == 7).all())


def torch_attention(c, q, n, t):
    """The definition in 64 bits on the GPU, for shapes that numpy takes long for."""
    hq, hkv = q.shape[1], c.hkv
    table = torch.from_numpy(R.numbers(np.arange(256, dtype=np.uint8), c.fmt)).cuda()
    k, v = (table[c.code[x][:, :n].long()] * c.scale[x].double().repeat_interleave(c.block, 1)[:, :n, None] for x in "kv")
    out = torch.empty(t, hq, D, dtype=torch.float64, device="cuda")
    see = torch.arange(n, device="cuda")[None] <= torch.arange(n - t, n, device="cuda")[:, None]
    for h in range(hq):
        x = (q[:, h].double() @ k[h // (hq // hkv)].T / np.sqrt(D)).masked_fill(~see, -float("inf"))
        out[:, h] = torch.softmax(x, 1) @ v[h // (hq // hkv)]
    return out


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,t,n,block", [(2, 2, 4150, 4200, 64), (32, 1, 300, 700, 16), (8, 1, 1, 70001, 128),
                                              (24, 8, 1, 40000, 32)])
def test_attention_of_many_rows_and_long_contexts(hq, hkv, t, n, block, fmt):
    g = torch.Generator(device="cuda").manual_seed(n)
    c = DeviceCache(fmt, block, n + 5, hkv)
    k, v = (torch.randn(n, hkv, D, generator=g, device="cuda").half() for _ in "kv")
    c.store(k, v, 0)
    q = torch.randn(t, hq, D, generator=g, device="cuda").half()
    got = attend(c, q, t, n).double().reshape(t, hq, D)
    want = torch_attention(c, q, n, t)
    # rounding of the result and of P: at most 2^-11 of the result and of sum p |v|, and |v| < 6
    assert float((got - want).abs().max()) <= 2.0 ** -11 * (6 + 6) + 2.0 ** -14
    rel = float((got - want).norm() / want.norm())
    assert rel <= 2.0 ** -11


@pytest.mark.parametrize("n", [1, 64, 1000, 1024, 1025, 20000])
def test_attention_workspace(n):
    """The size asked for is enough (and what lies behind it is not written), one byte less is refused, a workspace
    for n serves smaller n, and a null workspace gives the same bits."""
    g = torch.Generator(device="cuda").manual_seed(n)
    c = DeviceCache("e4m3", 128, n, 2)
    c.store(*(torch.randn(n, 2, D, generator=g, device="cuda").half() for _ in "kv"), 0)
    q = torch.randn(1, 8, D, generator=g, device="cuda").half()
    for with_acc in (False, True):
        need = E.kv8_attention_workspace(c.h, 8, 1, n, with_acc)
        w = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
        accs = [torch.zeros(2, n, device="cuda") if with_acc else None for _ in range(2)]
        a = attend(c, q, 1, n, acc=accs[0], ws=w[:need])
        assert bool((w[need:] == 0xAB).all())
        b = attend(c, q, 1, n, acc=accs[1], ws=None)
        assert torch.equal(a, b) and (not with_acc or torch.equal(accs[0], accs[1]))
        assert (need == 0) == (n <= 1024)  # one launch that joins through distributed shared memory
        if need:
            st = E.lib().ylm_k_kv8_attention(c.h, ptr(q), 8 * D, 8, 1, n, None, ptr(accs[0]), ptr(a), 8 * D, ptr(w),
                                             need - 1, stream())
            assert st == E.Status.INVALID_ARG and b"workspace" in E.lib().ylm_last_error()
        for m in {1, n // 2 or 1, max(1, n - 1), max(1, n - 65)}:
            assert E.kv8_attention_workspace(c.h, 8, 1, m, with_acc) <= need


def test_attention_workspace_of_every_smaller_length_fits():
    c = DeviceCache("e4m3", 16, 30000, 8)
    for hq, t in ((8, 1), (64, 1), (32, 7), (24, 100)):
        sizes = [E.kv8_attention_workspace(c.h, hq, t, n, a) for a in (0, 1) for n in range(t, 30000, 211)]
        half_ = len(sizes) // 2
        for part in (sizes[:half_], sizes[half_:]):
            assert part == sorted(part)


def test_attention_is_reproducible():
    rng = np.random.default_rng(2)
    c, _ = filled(rng, "e4m3", 32, 5000, 8, 4999, 0.3)
    q = half(rng.standard_normal((4, 32, D)))
    runs = []
    for _ in range(3):
        acc = torch.zeros(8, 5000, device="cuda")
        runs.append((attend(c, q, 4, 4999, acc=acc), acc))
    for o, a in runs[1:]:
        assert torch.equal(o, runs[0][0]) and torch.equal(a, runs[0][1])


# ---------------------------------------------------------------- eviction


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hkv,n,keep,sink,recent,block", [
    (1, 1, 1, 0, 0, 16), (2, 2, 1, 1, 0, 16), (2, 2, 1, 0, 1, 16), (3, 100, 37, 4, 8, 16), (8, 515, 200, 0, 0, 32),
    (2, 1000, 999, 3, 100, 64), (2, 1000, 1000, 0, 0, 128), (4, 700, 64, 32, 32, 128), (1, 5000, 2047, 4, 1024, 64),
    (2, 1025, 1, 0, 0, 16), (2, 300, 0, 0, 0, 16), (1, 0, 0, 0, 0, 16), (1, 2048, 129, 129, 0, 32),
    (2, 4097, 2000, 4, 100, 64), (1, 9000, 9000, 0, 9000, 16), (2, 12289, 5000, 300, 4500, 32),
    (1, 40000, 15001, 4, 9000, 128), (3, 33333, 100, 0, 0, 64)])
def test_evict(hkv, n, keep, sink, recent, block, fmt):
    rng = np.random.default_rng(n + keep)
    cap, cap_d = n + 9, keep + 50
    c, ref = (filled(rng, fmt, block, cap, hkv, n) if n else
              (DeviceCache(fmt, block, cap, hkv), R.Cache(fmt, block, cap, hkv)))
    w = np.exp(3 * rng.standard_normal((hkv, cap))).astype(np.float32)
    w[:, rng.random(cap) < 0.3] = 0
    run_evict(c, ref, w, n, keep, sink, recent, cap_d)


def run_evict(c, ref, w, n, keep, sink, recent, cap_d):
    d = DeviceCache(c.fmt, c.block, cap_d, c.hkv)
    acc, acc_d = torch.from_numpy(w).cuda(), torch.full((c.hkv, cap_d), 5.0, device="cuda")
    kept = torch.full((c.hkv, keep + 1), -7, dtype=torch.int32, device="cuda").reshape(-1)
    evict(c, d, acc, acc_d, n, keep, sink, recent, kept)
    want, dref, acc_ref = ref.evict(w.astype(np.float64), n, keep, sink, recent, cap_d)
    np.testing.assert_array_equal(kept[:c.hkv * keep].cpu().numpy().reshape(c.hkv, keep), want)
    assert bool((kept[c.hkv * keep:] == -7).all())
    d.same_as(dref, keep)
    np.testing.assert_array_equal(acc_d.cpu().numpy(), acc_ref.astype(np.float32))


@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "special", "negative", "near"])
@pytest.mark.parametrize("size", [3001, 17000])
def test_evict_ties_and_special_weights(kind, size):
    rng = np.random.default_rng(4)
    n, hkv = size, 2
    c, ref = filled(rng, "e4m3", 16, n, hkv, n)
    w = np.zeros((hkv, n), np.float32)
    if kind == "equal":
        w[:] = 0.7
    elif kind == "few":
        w[:] = rng.integers(0, 3, (hkv, n))
    elif kind == "special":
        w[:] = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38], np.float32), (hkv, n))
        w[:, ::7] = -np.nan
    elif kind == "negative":
        w[:] = rng.standard_normal((hkv, n))
    elif kind == "near":  # differ in the last bits only
        w[:] = (np.float32(1.0).view(np.uint32) + rng.integers(0, 500, (hkv, n)).astype(np.uint32)).view(np.float32)
    for keep, sink, recent in ((n // 2, 4, 64), (10, 0, 0), (n - 101, 0, 1), (70, 6, 64), (n - 1, 2, 2)):
        run_evict(c, ref, w, n, keep, sink, recent, keep + 3)


def test_evict_scales_a_block_of_mixed_origin():
    # tokens of blocks 2^10 apart meet in one block
    rng = np.random.default_rng(5)
    for fmt in FMTS:
        n = 320
        k = rng.standard_normal((n, 1, D)) * np.exp2(rng.integers(-10, 4, 20)).repeat(16)[:, None, None]
        k[32:48] = 0
        k = k.astype(np.float16)
        c, ref = DeviceCache(fmt, 16, n, 1), R.Cache(fmt, 16, n, 1)
        c.store(half(k), half(k[::-1].copy()), 0)
        ref.store(k.astype(np.float64), k[::-1].astype(np.float64), 0)
        run_evict(c, ref, rng.random((1, n)).astype(np.float32), n, 70, 2, 5, 100)


# ---------------------------------------------------------------- large offsets, streams, graphs


def test_offsets_beyond_32_bits():
    """A last KV head that starts 4.4 GB into the cache: store, attention and eviction address it."""
    hkv, cap, n = 8, 4_915_200, 200
    rng = np.random.default_rng(8)
    c = DeviceCache.__new__(DeviceCache)
    c.fmt, c.block, c.cap, c.hkv = "e4m3", 128, cap, hkv
    c.code = {x: torch.zeros(hkv, cap, D, dtype=torch.uint8, device="cuda") for x in "kv"}
    c.scale = {x: torch.zeros(hkv, cap // 128, device="cuda") for x in "kv"}
    c.h = E.kv8_cache(ptr(c.code["k"]), ptr(c.code["v"]), ptr(c.scale["k"]), ptr(c.scale["v"]), "e4m3", 128, cap, hkv)
    assert (hkv - 1) * cap * D > 2 ** 32
    ref = R.Cache("e4m3", 128, 300, hkv)
    k, v = rows(rng, n, hkv, 0.4), rows(rng, n, hkv, 0.4)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    for x in "kv":
        np.testing.assert_array_equal(R.numbers(c.code[x][:, :n].cpu().numpy(), "e4m3"), ref.num[x][:, :n])
    q = rng.standard_normal((2, 16, D)).astype(np.float16)
    acc = torch.zeros(hkv, cap, device="cuda")
    out = attend(c, half(q), 2, n, None, acc)
    want, w, pv, mag = R.attention(q.astype(np.float64), ref.values("k", n), ref.values("v", n), 2, np.zeros(n, bool))
    tol, dp = bounds(want, pv, mag, acc)
    assert np.all(np.abs(out.float().cpu().numpy().reshape(want.shape) - want) <= tol)
    d = DeviceCache("e4m3", 128, 90, hkv)
    acc_d, kept = torch.empty(hkv, 90, device="cuda"), torch.empty(hkv, 80, dtype=torch.int32, device="cuda")
    evict(c, d, acc, acc_d, n, 80, 4, 16, kept)
    kref, dref, _ = ref.evict(acc[:, :n].cpu().numpy().astype(np.float64), n, 80, 4, 16, 90)
    np.testing.assert_array_equal(kept.cpu().numpy(), kref)
    for x in "kv":
        np.testing.assert_array_equal(d.numbers(x)[:, :80], dref.num[x][:, :80])
    # the far end of the cache: the last slots of the last head
    c.store(half(k[:3]), half(v[:3]), cap - 3)
    ref2 = R.Cache("e4m3", 128, 128, hkv)
    ref2.scale["k"][:, 0] = 0
    ref2.store(k[:3].astype(np.float64), v[:3].astype(np.float64), 125)
    for x in "kv":
        np.testing.assert_array_equal(R.numbers(c.code[x][:, cap - 3:].cpu().numpy(), "e4m3"), ref2.num[x][:, 125:])


def step(c, d, q, k, v, slot, acc, acc_d, out, kept, ws, s):
    """A step and an eviction, all on stream s."""
    c.store(k, v, slot, s)
    attend(c, q, q.shape[0], slot + k.shape[0], acc=acc, out=out, ws=ws, s=s)
    evict(c, d, acc, acc_d, slot + k.shape[0], kept.shape[1], 2, 4, kept, s)


@pytest.mark.parametrize("n", [700, 2500])
@pytest.mark.parametrize("own_ws", [True, False])
def test_side_stream_and_captured_graphs(own_ws, n):
    """The three calls on a side stream, and captured in two graphs that are replayed together, each with its own
    buffers, give what the same calls give one after another."""
    rng = np.random.default_rng(9)
    hkv, hq, t = 2, 8, 3
    sides = []
    for _ in range(2):
        k0, v0 = half(rows(rng, n, hkv)), half(rows(rng, n, hkv))
        new = [half(rows(rng, t, hkv)) for _ in range(2)]
        sides.append((k0, v0, new[0], new[1], half(rng.standard_normal((t, hq, D)))))

    def fresh(side):
        k0, v0, k, v, q = side
        c, d = DeviceCache("e4m3", 32, n + t, hkv), DeviceCache("e4m3", 32, 400, hkv)
        c.store(k0, v0, 0)
        need = E.kv8_attention_workspace(c.h, hq, t, n + t, True)
        assert (need > 0) == (n > 1024)
        return [c, d, q, k, v, n, torch.zeros(hkv, n + t, device="cuda"), torch.zeros(hkv, 400, device="cuda"),
                torch.zeros(t, hq * D, dtype=torch.float16, device="cuda"),
                torch.zeros(hkv, 300, dtype=torch.int32, device="cuda"),
                torch.empty(need, dtype=torch.uint8, device="cuda") if own_ws else None]

    def results(a):
        return [a[8], a[6], a[9], a[7], a[1].code["k"][:, :300], a[1].code["v"][:, :300], a[1].scale["k"][:, :10]]

    want = []
    for side in sides:
        a = fresh(side)
        step(*a, stream())
        torch.cuda.synchronize()
        want.append([x.clone() for x in results(a)])
    side_stream = torch.cuda.Stream()
    a = fresh(sides[0])
    torch.cuda.synchronize()
    step(*a, side_stream.cuda_stream)
    side_stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(results(a), want[0]))

    graphs, states = [], []
    for side in sides:
        a = fresh(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(*a, stream())
        graphs.append(g)
        states.append(a)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for a in states:
            a[6].zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, w in zip(states, want):
            assert all(torch.equal(x, y) for x, y in zip(results(a), w))


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("prompt,budget,cap", [(517, 256, 640), (1500, 1100, 1536)])
def test_a_long_request_on_a_fixed_budget(fmt, prompt, budget, cap):
    """A prompt is stored, its last tokens' attention weighs the slots, the cache is evicted to its budget, decode
    steps follow behind the kept slots, it is evicted again into the first cache's buffers, and the request's
    logits are scored. Every step is held to the definitions in 64 bits."""
    rng = np.random.default_rng(12)
    hq, hkv, block = 8, 2, 32
    c, d = DeviceCache(fmt, block, cap, hkv), DeviceCache(fmt, block, cap, hkv)
    ref = R.Cache(fmt, block, cap, hkv)
    k, v = rows(rng, prompt, hkv, 0.4), rows(rng, prompt, hkv, 0.4)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    acc, acc_d = torch.zeros(hkv, cap, device="cuda"), torch.zeros(hkv, cap, device="cuda")
    q = rng.standard_normal((16, hq, D)).astype(np.float16)
    check_attention(c, ref, q, 16, prompt, None, acc)
    n, last = prompt, None
    for _ in range(2):
        kept = torch.zeros(hkv, budget, dtype=torch.int32, device="cuda")
        evict(c, d, acc, acc_d, n, budget, 4, 64, kept)
        want, ref, acc_ref = ref.evict(acc.cpu().numpy().astype(np.float64), n, budget, 4, 64, cap)
        np.testing.assert_array_equal(kept.cpu().numpy(), want)
        np.testing.assert_array_equal(acc_d.cpu().numpy(), acc_ref.astype(np.float32))
        c, d, acc, acc_d, n = d, c, acc_d, acc, budget
        for _ in range(40):
            k, v = rows(rng, 1, hkv, 0.4), rows(rng, 1, hkv, 0.4)
            c.store(half(k), half(v), n)
            ref.store(k.astype(np.float64), v.astype(np.float64), n)
            n += 1
            q = rng.standard_normal((1, hq, D)).astype(np.float16)
            last = check_attention(c, ref, q, 1, n, None, acc)
    # the output projection to a small vocabulary, and the answer's log probabilities
    vocab = 1000
    w = half(rng.standard_normal((vocab, hq * D)) * 0.3)
    logits = torch.empty(1, vocab, dtype=torch.float16, device="cuda")
    E.check(E.lib().ylm_k_gemm(ptr(last), ptr(w), 1, vocab, hq * D, ptr(logits), 1, stream()), "gemm")
    ids = logits.argmax(1)
    lp, top = torch.zeros(1, device="cuda"), torch.zeros(1, 3, device="cuda")
    top_ids = torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    E.check(E.lib().ylm_k_logprobs(ptr(logits), vocab, 1, vocab, ptr(ids), None, 3, ptr(lp), None, ptr(top_ids),
                                   ptr(top), stream()), "logprobs")
    x = logits.cpu().numpy().astype(np.float64)
    ref_lp, _, _, _ = R.logprobs(x, np.ones(vocab, bool))
    np.testing.assert_array_equal(top_ids.cpu().numpy()[0], R.top(x[0], np.ones(vocab, bool), 3))
    np.testing.assert_allclose(top.cpu().numpy()[0], ref_lp[0][top_ids.cpu().numpy()[0]], rtol=1e-5, atol=1e-5)
    assert float(lp[0]) == float(top[0, 0])


def test_a_failed_call_does_not_fail_the_next_one():
    # a workspace that no device has is refused by the allocator, before any launch
    c, ref = DeviceCache("e4m3", 16, 32, 1), R.Cache("e4m3", 16, 32, 1)
    q = torch.zeros(1, 8 * 128 * D, dtype=torch.float16, device="cuda")
    big = E.kv8_cache(ptr(c.code["k"]), ptr(c.code["v"]), ptr(c.scale["k"]), ptr(c.scale["v"]), "e4m3", 16, 1 << 30, 8)
    assert E.kv8_attention_workspace(big, 8 * 128, 1, 1 << 30, True) > 1 << 42
    acc = torch.zeros(32, device="cuda")
    for _ in range(2):
        assert E.lib().ylm_k_kv8_attention(big, ptr(q), q.stride(0), 8 * 128, 1, 1 << 30, None, ptr(acc), ptr(q),
                                           q.stride(0), None, 0, stream()) == E.Status.CUDA_ERROR
    k = rows(np.random.default_rng(0), 20, 1)
    c.store(half(k), half(k), 0)
    ref.store(k.astype(np.float64), k.astype(np.float64), 0)
    c.same_as(ref, 20)
    # nor a launch elsewhere in the library
    assert E.lib().ylm_k_kv8_attention(big, ptr(q), q.stride(0), 8 * 128, 1, 1 << 30, None, ptr(acc), ptr(q),
                                       q.stride(0), None, 0, stream()) == E.Status.CUDA_ERROR
    a = torch.ones(130, 128, dtype=torch.float16, device="cuda")
    o = torch.zeros(130, 130, dtype=torch.float16, device="cuda")
    E.check(E.lib().ylm_k_gemm(ptr(a), ptr(a), 130, 130, 128, ptr(o), 1, stream()), "gemm")
    assert bool((o == 128).all())


# ---------------------------------------------------------------- values and scores far apart


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,n", [(1, 20), (3, 22), (1, 1100), (2, 1200)])
@pytest.mark.parametrize("hq", [2, 8, 24])
def test_attention_of_small_values_beside_a_block_of_large_ones(fmt, t, n, hq):
    """A block with one channel of 30000 and small values elsewhere, whose scales are 2^24 apart: the other channels
    come from the small values alone, and keep their digits."""
    rng = np.random.default_rng(n + hq)
    hkv = 2
    k = rng.standard_normal((n, hkv, D)).astype(np.float16)
    v = (1 + rng.random((n, hkv, D))) * 2.0 ** -11
    v[:16] = 0
    v[:16, :, 0] = rng.choice([-30000, 30000], (16, hkv))
    v = v.astype(np.float16)
    c, ref = DeviceCache(fmt, 16, n, hkv), R.Cache(fmt, 16, n, hkv)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    scale = ref.scale["v"]
    assert np.all(scale[:, 0] / scale[:, 1] >= 2.0 ** 23)
    hidden = np.zeros(n, bool)
    hidden[18:n - t] = True
    q = (rng.standard_normal((t, hq, D)) * 0.2).astype(np.float16)
    check_attention(c, ref, q, t, n, hidden, torch.zeros(hkv, n, device="cuda"))
    check_attention(c, ref, q, t, n)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [12, 1100])
@pytest.mark.parametrize("order", ["first", "last"])
def test_attention_of_large_values_behind_a_slot_that_takes_the_weight(fmt, n, order):
    """One slot of value 0 takes all but about 2^-24 of the weight; what is left meets values of 20000."""
    rng = np.random.default_rng(n)
    hkv, hq = 1, 4
    at = 0 if order == "first" else 11
    q = np.repeat(rng.standard_normal((1, 1, D)), hq, 1).astype(np.float16)
    k = (rng.standard_normal((n, hkv, D)) * 0.05).astype(np.float16)
    v = (rng.standard_normal((n, hkv, D)) * 8000).astype(np.float16)
    v[at] = 0
    length = float((q[0, 0].astype(np.float64) ** 2).sum())
    k[at, 0] = (q[0, 0].astype(np.float64) * (15.8 * np.sqrt(D) / length)).astype(np.float16)
    c, ref = DeviceCache(fmt, 16, n, hkv), R.Cache(fmt, 16, n, hkv)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    hidden = np.zeros(n, bool)
    hidden[12:] = True
    out, _, _, _ = R.attention(q.astype(np.float64), ref.values("k", n), ref.values("v", n), 1, hidden)
    assert 2.0 ** -15 < np.abs(out).max() < 2.0 ** -5
    check_attention(c, ref, q, 1, n, hidden, torch.zeros(hkv, n, device="cuda"))




@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,n,hq", [(1, 300, 8), (1, 1300, 8), (4, 500, 16), (6, 1400, 24)])
@pytest.mark.parametrize("seed", range(4))
def test_attention_of_values_at_random_scales(fmt, t, n, hq, seed):
    """Every block of values at a scale of its own, up to 2^26 apart, some blocks of zeros, some slots hidden; each
    block uses a few dimensions only, so that small values stand alone in many."""
    rng = np.random.default_rng(100 * n + seed)
    hkv, nb = 2, -(-n // 16)
    k = rng.standard_normal((n, hkv, D)).astype(np.float16)
    size = np.exp2(rng.uniform(-14, 12, (nb, hkv)))
    size[rng.random((nb, hkv)) < 0.1] = 0
    v = rng.standard_normal((n, hkv, D)) * np.repeat(size, 16, 0)[:n, :, None]
    v *= np.repeat(rng.random((nb, hkv, D)) < 0.1, 16, 0)[:n]
    v = v.astype(np.float16)
    c, ref = DeviceCache(fmt, 16, n, hkv), R.Cache(fmt, 16, n, hkv)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    q = (rng.standard_normal((t, hq, D)) * 0.5).astype(np.float16)
    check_attention(c, ref, q, t, n, None, torch.zeros(hkv, n, device="cuda"))
    check_attention(c, ref, q, t, n, rng.random(n) < 0.7)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,n,hq", [(1, 40, 2), (1, 300, 8), (1, 1300, 8), (3, 500, 16), (2, 1300, 24)])
@pytest.mark.parametrize("size", [500, 1500, 2500, 4000, 6000, 10000, 20000])
def test_attention_of_the_largest_scores(fmt, t, n, hq, size):
    """Scores up to 10^10, where FP32 steps by octaves and more: one slot takes each row, its value is the result, and
    the row's weight adds up to one."""
    rng = np.random.default_rng(n + size)
    hkv = 2
    k = np.clip(rng.standard_normal((n, hkv, D)) * size, -65504, 65504).astype(np.float16)
    v = (rng.standard_normal((n, hkv, D)) * np.exp2(rng.integers(-8, 8, -(-n // 16))).repeat(16)[:n, None, None])
    v = v.astype(np.float16)
    c, ref = DeviceCache(fmt, 16, n, hkv), R.Cache(fmt, 16, n, hkv)
    c.store(half(k), half(v), 0)
    ref.store(k.astype(np.float64), v.astype(np.float64), 0)
    q = np.clip(rng.standard_normal((t, hq, D)) * size, -65504, 65504).astype(np.float16)
    acc = torch.zeros(hkv, n, device="cuda")
    got = attend(c, half(q), t, n, acc=acc).float().cpu().numpy().astype(np.float64).reshape(t, hq, D)
    same = attend(c, half(q), t, n).float().cpu().numpy().astype(np.float64).reshape(t, hq, D)
    kv, vv = ref.values("k", n), ref.values("v", n)
    G, weight, sure = hq // hkv, np.zeros((hkv, n)), np.ones(hkv, bool)
    for h in range(hq):
        for i in range(t):
            m, g = n - t + i + 1, h // G
            x = kv[g, :m] @ q[i, h].astype(np.float64) / np.sqrt(D)
            err = 2.0 ** -17 * (np.abs(kv[g, :m]) @ np.abs(q[i, h].astype(np.float64))).max() / np.sqrt(D)
            best = int(x.argmax())
            weight[g, best] += 1
            if np.partition(x, -2)[-2] + err + 21 < x[best]:  # by more than the sums' rounding and 30 octaves
                lo = hi = vv[g, best]
            else:
                lo, hi, sure[g] = vv[g, :m].min(0), vv[g, :m].max(0), False
            for out in (got, same):
                assert np.all(out[i, h] >= lo - EPS16 * np.abs(lo) * 2 - 2.0 ** -24)
                assert np.all(out[i, h] <= hi + EPS16 * np.abs(hi) * 2 + 2.0 ** -24)
    assert sure.any()
    acc = acc.cpu().numpy()
    np.testing.assert_allclose(acc[sure], weight[sure], rtol=2.0 ** -12, atol=2.0 ** -12)
    np.testing.assert_allclose(acc.sum(1), weight.sum(1), rtol=2.0 ** -12)
