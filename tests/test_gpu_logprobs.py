"""Log probabilities of rows of FP16 logits on the GPU, through the C ABI, against their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

import kv8_reference as R
from yalama_b200 import engine as E

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ptr(t):
    return None if t is None else t.data_ptr()


def bits(masked):
    w = np.zeros((masked.size + 31) // 32, np.uint32)
    for i in np.nonzero(masked)[0]:
        w[i >> 5] |= np.uint32(1) << np.uint32(i & 31)
    return torch.from_numpy(w.view(np.int32)).cuda()


def run(x, ids, n_top, masked=None, ld=None, shift=0, want=("logprob", "entropy"), s=None):
    """x [rows][vocab] float16; shift: the first logit's offset in halves from an aligned address."""
    rows, vocab = x.shape
    ld = vocab if ld is None else ld
    # what lies around the rows must not count
    buf = torch.full((shift + rows * ld + 64,), float("nan"), dtype=torch.float16, device="cuda")
    view = buf[shift:shift + rows * ld].reshape(rows, ld)
    view[:, :vocab] = torch.from_numpy(x).cuda()
    o = {"logprob": torch.full((rows + 1,), 7.0, device="cuda"), "entropy": torch.full((rows + 1,), 7.0, device="cuda"),
         "top_ids": torch.full((rows + 1, max(n_top, 1)), 7, dtype=torch.int64, device="cuda"),
         "top": torch.full((rows + 1, max(n_top, 1)), 7.0, device="cuda")}
    d_ids = torch.from_numpy(np.asarray(ids, np.int64)).cuda() if "logprob" in want else None
    E.check(E.lib().ylm_k_logprobs(ptr(view), ld, rows, vocab, ptr(d_ids), None if masked is None else ptr(bits(masked)),
                                   n_top, ptr(o["logprob"]) if "logprob" in want else None,
                                   ptr(o["entropy"]) if "entropy" in want else None, ptr(o["top_ids"]), ptr(o["top"]),
                                   torch.cuda.current_stream().cuda_stream if s is None else s), "logprobs")
    torch.cuda.synchronize()
    for name, t in o.items():  # nothing behind the last row
        assert bool((t[rows:] == 7).all()), name
        if name in ("logprob", "entropy") and name not in want or name.startswith("top") and not n_top:
            assert bool((t == 7).all()), name
    return {k: t[:rows].cpu().numpy() for k, t in o.items()}


def check(x, ids, n_top, masked=None, **kw):
    """z and the entropy's sum are sums of positive terms: a term takes an exponential (within 2^-21 of it), a thread
    adds at most vocab / 128 + 8 terms one after another and 64 partial sums follow, each addition off by at most
    2^-24 of the sum: rel = (vocab / 128 + 72) 2^-24 + 2^-21 of z. log1p and the subtractions add a few steps."""
    rows, vocab = x.shape
    seen = np.ones(vocab, bool) if masked is None else ~masked
    got = run(x, ids, n_top, masked, **kw)
    lp, ent, m, z = R.logprobs(x.astype(np.float64), seen)
    rel = (vocab / 128 + 72) * 2.0 ** -24 + 2.0 ** -21
    lz = np.log1p(z)

    def tol(v, r):
        return rel * z[r] / (1 + z[r]) + 2.0 ** -22 * (np.abs(v) + 2 * lz[r]) + 1e-37

    for r in range(rows):
        w = lp[r, ids[r]] if 0 <= ids[r] < vocab else -np.inf
        if np.isfinite(w):
            assert abs(got["logprob"][r] - w) <= tol(w, r), (r, got["logprob"][r], w)
        else:
            assert got["logprob"][r] == w
        assert abs(got["entropy"][r] - ent[r]) <= rel * (z[r] / (1 + z[r]) + 2 * ent[r]) + 2.0 ** -21 * ent[r] + 1e-37
        if n_top:
            want = R.top(x[r].astype(np.float64), seen, n_top)
            np.testing.assert_array_equal(got["top_ids"][r], want)
            for i, v in zip(want, got["top"][r]):
                assert v == -np.inf if i < 0 else abs(v - lp[r, i]) <= tol(lp[r, i], r)


@pytest.mark.parametrize("rows,vocab,n_top", [
    (1, 1, 0), (1, 1, 1), (1, 1, 64), (3, 2, 2), (2, 7, 7), (1, 8, 20), (5, 31, 5), (2, 63, 64), (2, 64, 64),
    (2, 65, 64), (4, 1000, 20), (1, 4095, 20), (1, 4096, 1), (3, 8191, 64), (2, 32768, 5), (1, 128256, 20),
    (1, 151936, 64), (3, 50257, 0), (17, 2049, 3), (40, 8200, 20), (160, 1024, 10), (300, 513, 33)])
def test_logprobs(rows, vocab, n_top):
    rng = np.random.default_rng(rows * 1000 + vocab)
    x = (rng.standard_normal((rows, vocab)) * rng.uniform(0.1, 6, (rows, 1))).astype(np.float16)
    check(x, rng.integers(0, vocab, rows), n_top)
    masked = rng.random(vocab) < 0.3
    check(x, rng.integers(0, vocab, rows), n_top, masked)
    # rows that start anywhere, with room behind each
    check(x, x.astype(np.float32).argmax(1), n_top, masked, ld=vocab + 3, shift=int(rng.integers(1, 8)))


@pytest.mark.parametrize("vocab", [100, 3000, 40000])
@pytest.mark.parametrize("order", ["up", "down", "same", "two", "zeros", "steps"])
def test_orders_and_ties(vocab, order):
    x = {"up": np.linspace(-20, 20, vocab), "down": np.linspace(20, -20, vocab), "same": np.full(vocab, 1.5),
         "two": np.where(np.arange(vocab) % 3 == 1, 2.0, -1.0), "zeros": np.where(np.arange(vocab) % 2 == 1, 0.0, -0.0),
         "steps": np.floor(np.arange(vocab) / 50) % 7}[order].astype(np.float16)[None]
    for n_top in (1, 20, 64):
        check(x, [vocab // 2], n_top)
        check(x, [vocab - 1], n_top, np.arange(vocab) % 5 == 0)


@pytest.mark.parametrize("vocab", [9, 1000, 128256])
def test_certain_rows_keep_small_log_probabilities(vocab):
    # the likeliest id's log probability is -(vocab - 1) e^-gap, far below the step of 1
    for gap in (10, 18, 30, 60):
        x = np.full((2, vocab), -gap / 2, np.float16)
        x[0, vocab // 3] = gap / 2
        x[1, vocab - 1] = gap / 2
        check(x, [vocab // 3, 0], 3)
        got = run(x, [vocab // 3, vocab - 1], 1)
        assert np.all(got["logprob"] < 0) and np.all(got["entropy"] > 0)


def test_extreme_logits():
    x = np.full((4, 5000), -65504, np.float16)
    x[1, 7] = 65504
    x[2, ::2] = 65504
    x[3] = 65504
    check(x, [0, 7, 1, 4999], 9)


def test_rows_without_any_id():
    x = np.full((3, 700), -np.inf, np.float16)
    x[1] = 1.0
    for masked in (None, np.ones(700, bool)):
        got = run(x, [0, 5, -1], 4, masked)
        for r in range(3):
            if masked is None and r == 1:
                continue
            assert got["logprob"][r] == -np.inf and got["entropy"][r] == 0
            assert np.all(got["top_ids"][r] == -1) and np.all(got["top"][r] == -np.inf)
    # masked ids and ids outside the vocabulary have no probability
    masked = np.zeros(700, bool)
    masked[5] = True
    for i in (5, -1, 700, 2 ** 40, -2 ** 40):
        assert run(x[1:2], [i], 0, masked)["logprob"][0] == -np.inf


def test_minus_infinity_among_the_logits():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 2000)).astype(np.float16)
    x[0, :1990] = -np.inf
    x[1, 100:] = -np.inf
    x[2, 5] = -np.inf
    check(x, [1995, 3, 5], 20)


def test_nan_and_infinity():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 3000)).astype(np.float16)
    x[0, 1234] = np.nan
    x[1, 17] = np.inf
    x[2, 99] = -np.nan
    got = run(x, [5, 17, 99, 5], 3)
    for r in range(3):
        assert np.isnan(got["logprob"][r]) and np.isnan(got["entropy"][r]) and np.isnan(got["top"][r]).all()
    assert [got["top_ids"][r][0] for r in range(3)] == [1234, 17, 99]
    assert np.isfinite(got["logprob"][3])
    # masked, they do not count
    masked = np.zeros(3000, bool)
    masked[[1234, 17, 99]] = True
    check(x, [5, 6, 7, 8], 20, masked)


def test_outputs_that_are_not_wanted():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 500)).astype(np.float16)
    both = run(x, [1, 2], 3)
    for want in ((), ("logprob",), ("entropy",)):
        got = run(x, [1, 2], 3, want=want)
        np.testing.assert_array_equal(got["top"], both["top"])
        for name in want:
            np.testing.assert_array_equal(got[name], both[name])


def test_more_rows_than_a_grid_dimension():
    rng = np.random.default_rng(6)
    rows, vocab = 70001, 37
    x = rng.standard_normal((rows, vocab)).astype(np.float16)
    ids = rng.integers(0, vocab, rows)
    got = run(x, ids, 2)
    lp, ent, _, _ = R.logprobs(x.astype(np.float64), np.ones(vocab, bool))
    np.testing.assert_allclose(got["logprob"], lp[np.arange(rows), ids], rtol=1e-5, atol=1e-6)
    np.testing.assert_allclose(got["entropy"], ent, rtol=1e-5)
    best = np.argsort(-x.astype(np.float64), 1, kind="stable")[:, :2]
    np.testing.assert_array_equal(got["top_ids"], best)


def test_rows_beyond_32_bits():
    # the last row lies 4.3 G logits behind the first
    vocab, ld, rows = 1000, 1 << 27, 33
    rng = np.random.default_rng(4)
    buf = torch.empty(ld * (rows - 1) + vocab, dtype=torch.float16, device="cuda")
    x = rng.standard_normal((rows, vocab)).astype(np.float16)
    for r in range(rows):
        buf[r * ld:r * ld + vocab] = torch.from_numpy(x[r]).cuda()
    ids = torch.arange(rows, device="cuda")
    lp, ent = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    E.check(E.lib().ylm_k_logprobs(ptr(buf), ld, rows, vocab, ptr(ids), None, 0, ptr(lp), ptr(ent), None, None,
                                   torch.cuda.current_stream().cuda_stream), "logprobs")
    want, went, _, _ = R.logprobs(x.astype(np.float64), np.ones(vocab, bool))
    np.testing.assert_allclose(lp.cpu().numpy(), want[np.arange(rows), np.arange(rows)], rtol=1e-5)
    np.testing.assert_allclose(ent.cpu().numpy(), went, rtol=1e-5)


def test_side_stream_and_captured_graph():
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((3, 40000)).astype(np.float16)).cuda()
    ids = torch.tensor([1, 2, 3], device="cuda")

    def call(o, s):
        E.check(E.lib().ylm_k_logprobs(ptr(x), 40000, 3, 40000, ptr(ids), None, 20, ptr(o[0]), ptr(o[1]), ptr(o[2]),
                                       ptr(o[3]), s), "logprobs")

    def outs():
        return [torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"),
                torch.zeros(3, 20, dtype=torch.int64, device="cuda"), torch.zeros(3, 20, device="cuda")]

    want, got, cap = outs(), outs(), outs()
    torch.cuda.synchronize()
    call(want, torch.cuda.current_stream().cuda_stream)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(got, side.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(cap, torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, cap):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_engine_logprobs_of_a_generated_token():
    """ylm_logprobs after a prefill and after decode steps: the engine's own logits in 64 bits; masked ids left
    out on request; neither the logits nor the tokens that follow change."""
    from yalama_b200 import synth
    spec = synth.tiny_spec("qwen3")
    eng = E.Engine(None, E.config_from_spec(spec), init_seed=0)
    with pytest.raises(E.YlmError) as ei:
        eng.logprobs(0)
    assert ei.value.status == E.Status.NOT_READY
    prompt = synth.prompt_ids(0, 16, spec.vocab)
    plain = eng.generate(prompt, 8)["ids"]
    eng.set_sampling(greedy=True, masked_ids=[int(plain[1]), 3])
    eng.begin_infer()
    assert eng.infer(prompt)[0] == E.Status.OK
    token, ids = eng.sample(True), []
    rel = (spec.vocab / 128 + 72) * 2.0 ** -24 + 2.0 ** -21  # as in check()
    for step in range(8):
        x = eng.logits().astype(np.float64)[None]
        for masked in (False, True):
            seen = np.ones(spec.vocab, bool)
            if masked:
                seen[[int(plain[1]), 3]] = False
            lp, ent, _, z = R.logprobs(x, seen)
            got = eng.logprobs(token, 5, masked)
            tol = rel + 2.0 ** -21 * (20 + ent[0])
            if np.isfinite(lp[0, token]):
                assert abs(got["logprob"] - lp[0, token]) <= tol
            else:
                assert got["logprob"] == -np.inf
            assert abs(got["entropy"] - ent[0]) <= rel * (1 + 2 * ent[0]) + 2.0 ** -21 * ent[0]
            want = R.top(x[0], seen, 5)
            np.testing.assert_array_equal(got["top_ids"], want)
            assert np.all(np.abs(got["top_logprobs"] - lp[0, want]) <= tol)
        np.testing.assert_array_equal(eng.logits(), x[0].astype(np.float32))
        assert eng.logprobs(-1)["logprob"] == -np.inf and eng.logprobs(spec.vocab)["logprob"] == -np.inf
        ids.append(token)
        st, token = eng.decode(token, True)
        assert st == E.Status.OK
    assert ids == [int(i) for i in plain]
    for bad in (dict(n_top=65), dict(n_top=-1)):
        with pytest.raises(E.YlmError):
            eng.logprobs(0, **bad) if bad["n_top"] > 0 else E.check(
                E.lib().ylm_logprobs(eng._h, 0, -1, 0, None, None, None, None), "x")
    eng.close()


def test_engine_logprobs_after_a_token_loop():
    """After ylm_generate the log probabilities are those of the last token it read, or refused where the loop had
    run a step past an EOS, whose logits belong to no token of the request."""
    from yalama_b200 import synth
    spec = synth.tiny_spec("llama", tied=False, rope_theta=5e5, heads=8, kv_heads=2)
    eng, ref = (E.Engine(None, E.config_from_spec(spec), init_seed=0) for _ in range(2))
    for e in (eng, ref):
        e.set_sampling(greedy=True)
    prompt = synth.prompt_ids(12, 32, spec.vocab)
    ids = [int(t) for t in eng.generate(prompt, 20)["ids"]]
    stop = next(i for i in range(3, len(ids) - 1) if ids[i] not in ids[:i])

    def want(count):
        """The log probabilities that token `count` was chosen by."""
        ref.begin_infer()
        ref.infer(prompt)
        for t in ids[:count]:
            ref.infer([t])
        return ref.logprobs(ids[count], 5)

    def same(a, b):
        assert a["logprob"] == b["logprob"] and a["entropy"] == b["entropy"]
        np.testing.assert_array_equal(a["top_ids"], b["top_ids"])
        np.testing.assert_array_equal(a["top_logprobs"], b["top_logprobs"])

    # the loop ends at max_new
    for count in (1, 2, 7):
        eng.generate(prompt, count)
        same(eng.logprobs(ids[count - 1], 5), want(count - 1))
    # at an EOS that is also the last token allowed: no step ran past it
    r = eng.generate(prompt, stop + 1, eos_ids=[ids[stop]])
    assert [int(t) for t in r["ids"]] == ids[:stop]
    same(eng.logprobs(ids[stop], 5), want(stop))
    # at an EOS with another step on its way
    r = eng.generate(prompt, 20, eos_ids=[ids[stop]])
    assert [int(t) for t in r["ids"]] == ids[:stop]
    with pytest.raises(E.YlmError) as ei:
        eng.logprobs(ids[stop], 5)
    assert ei.value.status == E.Status.NOT_READY
    # the next step has logits of its own
    eng.infer([ids[stop]])
    same(eng.logprobs(ids[stop + 1], 5), want(stop + 1))
    eng.generate(prompt, 20, eos_ids=[ids[stop]])
    eng.decode(ids[stop], True)
    same(eng.logprobs(ids[stop + 1], 5), want(stop + 1))
    eng.generate(prompt, 4)
    same(eng.logprobs(ids[3], 5), want(3))
    eng.close()
    ref.close()


def test_engine_logprobs_after_a_failed_step():
    """A step whose bounded wait ran out leaves logits of no token; the next request has its own."""
    from yalama_b200 import synth
    spec = synth.tiny_spec("llama", tied=False, rope_theta=5e5, heads=8, kv_heads=2)
    eng = E.Engine(None, E.config_from_spec(spec), init_seed=0, wait_limit_us=2000)
    prompt = synth.prompt_ids(13, 24, spec.vocab)
    eng.begin_infer()
    eng.infer(prompt)
    want = eng.logprobs(5, 3)
    eng.debug_drop_output(0)
    with pytest.raises(E.YlmError) as ei:
        eng.infer([5])
    assert ei.value.status == E.Status.DEVICE_TIMEOUT
    eng.debug_drop_output(-1)
    with pytest.raises(E.YlmError) as ei:
        eng.logprobs(5, 3)
    assert ei.value.status == E.Status.NOT_READY
    eng.begin_infer()
    eng.infer(prompt)
    got = eng.logprobs(5, 3)
    assert got["logprob"] == want["logprob"] and got["entropy"] == want["entropy"]
    eng.close()


# ---------------------------------------------------------------- special values in one CTA's part of a row

PARTS = [(3000, 1), (20001, 2), (40000, 4), (131077, 8)]  # ids, CTAs a row (one to four rows)


def part(vocab, parts, i):
    """The ids well inside part i of a row."""
    per = vocab // parts
    return slice(i * per + 16, (i + 1) * per - 16)


@pytest.mark.parametrize("vocab,parts", PARTS)
def test_parts_without_ids(vocab, parts):
    """Whole parts that are -inf or masked beside parts that are not, and fewer open ids than alternatives."""
    rng = np.random.default_rng(vocab)
    for i in range(parts):
        own = part(vocab, parts, i)
        x = rng.standard_normal((3, vocab)).astype(np.float16)
        x[0, own] = -np.inf                       # one part has next to no id
        x[1, :own.start], x[1, own.stop:] = -np.inf, -np.inf  # only one has
        x[2] = -np.inf                            # seven ids, all in one
        few = np.sort(rng.choice(np.arange(own.start, own.stop), 7, replace=False))
        x[2, few] = rng.standard_normal(7) * 3
        for n_top in (1, 20, 64):
            check(x, [vocab - 1, own.start + 3, few[2]], n_top)
        masked = np.ones(vocab, bool)             # the same by a mask
        masked[few] = False
        y = rng.standard_normal((2, vocab)).astype(np.float16)
        check(y, [few[0], (few[0] + 1) % vocab], 20, masked)
        check(y, [few[6], few[1]], 20, masked, ld=vocab + 5, shift=3)
        check(y, [few[0], own.start], 20, ~masked)
        masked = np.zeros(vocab, bool)
        masked[own] = True
        check(y, [own.start, vocab - 1], 20, masked)


@pytest.mark.parametrize("vocab,parts", PARTS)
def test_parts_with_nan_or_infinity(vocab, parts):
    rng = np.random.default_rng(vocab + 1)
    for i in range(parts):
        own = part(vocab, parts, i)
        x = rng.standard_normal((4, vocab)).astype(np.float16)
        at = own.start + 7
        x[0, at], x[1, at], x[2, at] = np.nan, np.inf, -np.nan
        x[2, vocab - 2] = np.nan  # two: the lower id first
        got = run(x, [5, at, 9, 5], 20)
        for r in range(3):
            assert np.isnan(got["logprob"][r]) and np.isnan(got["entropy"][r]) and np.isnan(got["top"][r]).all()
        assert got["top_ids"][0][0] == at and got["top_ids"][1][0] == at
        assert list(got["top_ids"][2][:2]) == [at, vocab - 2]
        rest = np.where(np.isnan(x[0]), -np.inf, x[0]).astype(np.float64)
        np.testing.assert_array_equal(got["top_ids"][0][1:], R.top(rest, np.ones(vocab, bool), 19))
        masked = np.zeros(vocab, bool)
        masked[[at, vocab - 2]] = True
        check(x, [5, 6, 9, 8], 20, masked)


@pytest.mark.parametrize("vocab,parts", PARTS)
def test_parts_of_the_lowest_and_the_highest_values(vocab, parts):
    rng = np.random.default_rng(vocab + 2)
    for i in range(parts):
        own = part(vocab, parts, i)
        x = rng.standard_normal((4, vocab)).astype(np.float16)
        x[0, own] = -65504
        x[1] = -65504
        x[1, own] = -np.inf
        x[2] = -65504
        x[2, own.start + 5] = -65472
        x[3, own] = 65504
        check(x, [own.start, 0, own.start + 5, own.start + 9], 20)


@pytest.mark.parametrize("vocab,parts", PARTS)
def test_rows_of_several_parts_without_any_id(vocab, parts):
    for masked in (None, np.ones(vocab, bool)):
        x = np.full((2, vocab), -np.inf if masked is None else 1.0, np.float16)
        got = run(x, [0, vocab - 1], 20, masked)
        assert np.all(got["logprob"] == -np.inf) and np.all(got["entropy"] == 0)
        assert np.all(got["top_ids"] == -1) and np.all(got["top"] == -np.inf)


@pytest.mark.parametrize("vocab", [3000017, 20000003])
def test_vocabularies_beyond_any_model(vocab):
    """One row, eight CTAs: a thread adds vocab / 4096 terms to a sum, and 72 additions join the sums."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(1, vocab, generator=g, device="cuda") * 2).half()
    ids = torch.tensor([vocab - 1], device="cuda")
    lp, ent = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    top_ids, top = torch.zeros(1, 20, dtype=torch.int64, device="cuda"), torch.zeros(1, 20, device="cuda")
    E.check(E.lib().ylm_k_logprobs(ptr(x), vocab, 1, vocab, ptr(ids), None, 20, ptr(lp), ptr(ent), ptr(top_ids),
                                   ptr(top), torch.cuda.current_stream().cuda_stream), "logprobs")
    want = torch.log_softmax(x.double(), 1)
    went = -(want.exp() * want).sum(1)
    rel = (vocab / 4096 + 72) * 2.0 ** -24 + 2.0 ** -21
    tol = rel + 2.0 ** -21 * 40  # log probabilities of at most 40
    assert abs(float(lp) - float(want[0, -1])) <= tol
    assert abs(float(ent) - float(went)) <= rel * (1 + 2 * float(went)) + 2.0 ** -21 * float(went)
    best = torch.sort(x[0].float(), descending=True, stable=True).indices[:20]
    assert torch.equal(top_ids[0], best)
    assert float((top[0].double() - want[0, best]).abs().max()) <= tol


def test_engine_logprobs_refuses_bad_counts():
    """Refused for the count alone: every pointer is good."""
    from yalama_b200 import synth
    spec = synth.tiny_spec("llama")
    eng = E.Engine(None, E.config_from_spec(spec), init_seed=0)
    eng.begin_infer()
    eng.infer(synth.prompt_ids(0, 8, spec.vocab))
    lp, ent = ctypes.c_float(), ctypes.c_float()
    ids, top = np.zeros(128, np.int64), np.zeros(128, np.float32)

    def call(n_top, i=ids, t=top):
        return E.lib().ylm_logprobs(eng._h, 0, n_top, 0, ctypes.byref(lp), ctypes.byref(ent),
                                    None if i is None else E._ptr(i, ctypes.c_int64),
                                    None if t is None else E._ptr(t, ctypes.c_float))

    for n_top in (-1, -2 ** 31, 65, 2 ** 31 - 1):
        assert call(n_top) == E.Status.INVALID_ARG
    assert call(1, None) == E.Status.INVALID_ARG and call(1, ids, None) == E.Status.INVALID_ARG
    assert call(64) == E.Status.OK and call(0, None, None) == E.Status.OK
    eng.close()
