"""Model-level parity on the GPU: the engine's token loop (prefill, decode,
sampling, KV-cache state machine) against the oracle's FP16-storage forward on
the same seeded weights, through the C ABI."""
import ctypes
import json
import os
import time

import numpy as np
import pytest

from yalama_b200 import engine as E
from yalama_b200 import synth
from oracle.model import OracleModel
from oracle import sampler as S
from oracle.numerics import sampler_uniform

pytestmark = pytest.mark.gpu

GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")
# the parity bar: logits within max-abs 2e-2 of the reference FP16 path
LOGIT_TOL = 2e-2
# greedy ids may differ only where the top-2 logit gap is below this
TIE_GAP = 1e-2

FAMILIES = {
    "qwen3": dict(model_type="qwen3"),
    "qwen2": dict(model_type="qwen2", tied=False),
    "llama": dict(model_type="llama", tied=False, rope_theta=5e5, heads=8, kv_heads=2),
    "mistral": dict(model_type="mistral", tied=False, heads=2, kv_heads=2),
    "llama_g8": dict(model_type="llama", tied=True, hidden=512, heads=16, kv_heads=2, intermediate=1024),
}


def make(kw, seed=0, snapshot=None, tmp=None, through_bf16=False, **opts):
    spec = synth.tiny_spec(**kw)
    snap = None
    if snapshot:
        snap = synth.write_snapshot(str(tmp), spec, seed=seed, dtype=snapshot, through_bf16=through_bf16)
    eng = E.Engine(snap, E.config_from_spec(spec), init_seed=seed, **opts)
    return spec, eng


def top2_gap(lg):
    s = np.sort(lg.astype(np.float64))
    return s[-1] - s[-2]


def run_teacher_forced(eng, orc, prompt, steps):
    """Prefill + decode `steps` tokens, feeding the oracle's greedy ids to both."""
    eng.begin_infer()
    orc.begin_infer()
    ids = list(prompt)
    worst = 0.0
    mismatch = 0
    for step in range(steps + 1):
        st, _ = eng.infer(ids)
        assert st == E.Status.OK
        so, lo = orc.infer(ids)
        assert so == 0
        lg = eng.logits()
        worst = max(worst, float(np.max(np.abs(lg - lo))))
        gid, oid = S.greedy(lg), S.greedy(lo)
        if gid != oid:
            assert top2_gap(lo) < TIE_GAP, (step, gid, oid, top2_gap(lo))
            mismatch += 1
        ids = [oid]
    return worst, mismatch


@pytest.mark.parametrize("persistent", [0, 1])
@pytest.mark.parametrize("fam", sorted(FAMILIES))
def test_family_logits_match_oracle(fam, persistent):
    spec, eng = make(FAMILIES[fam], decode_persistent=persistent)
    orc = OracleModel(spec, synth.model_weights(spec, 0), mode="f16", kv_gb=2)
    prompt = synth.prompt_ids(0, 24, spec.vocab)
    worst, _ = run_teacher_forced(eng, orc, prompt, 12)
    print(f"{fam}: max |logit diff| = {worst:.3e}")
    assert worst < LOGIT_TOL


@pytest.mark.parametrize("fam", ["llama", "qwen3"])
def test_split_attention_kernel_logits_match_oracle(fam):
    # the split-K decode attention (global partials, last-CTA combine), the
    # path where cluster launches are unavailable, in both decode paths
    with E.split_attention():
        for persistent in (0, 1):
            spec, eng = make(FAMILIES[fam], decode_persistent=persistent)
            orc = OracleModel(spec, synth.model_weights(spec, 0), mode="f16", kv_gb=2)
            prompt = synth.prompt_ids(9, 700, spec.vocab)
            worst, _ = run_teacher_forced(eng, orc, prompt, 6)
            eng.close()
            assert worst < LOGIT_TOL, (persistent, worst)


def test_snapshot_load_equals_random_init(tmp_path):
    """The loader (pinned row bands, BF16 / F32 converted on the device) gives
    the weights bit for bit: F16 and F32 shards of the generator's values load
    as the random init does, and BF16 shards load as an F16 snapshot of the
    same values rounded to BF16 (qwen2: QKV biases, untied lm_head)."""
    kw = FAMILIES["qwen2"]
    spec, a = make(kw)
    _, b = make(kw, snapshot="F16", tmp=tmp_path / "f16")
    _, c = make(kw, snapshot="BF16", tmp=tmp_path / "bf16")
    _, d = make(kw, snapshot="F32", tmp=tmp_path / "f32")
    _, e = make(kw, snapshot="F16", tmp=tmp_path / "f16_of_bf16", through_bf16=True)
    prompt = synth.prompt_ids(1, 16, spec.vocab)
    outs = []
    for eng in (a, b, c, d, e):
        eng.begin_infer()
        st, _ = eng.infer(prompt)
        assert st == E.Status.OK
        outs.append(eng.logits())
    # the same FP16 weights through the counter-based generator and through the loader
    np.testing.assert_array_equal(outs[0], outs[1])
    np.testing.assert_array_equal(outs[0], outs[3])
    # BF16 shards decode to exactly the BF16-rounded values
    np.testing.assert_array_equal(outs[2], outs[4])
    # and those differ from the FP16 weights by BF16 rounding only: close, not equal
    assert np.max(np.abs(outs[0] - outs[2])) < 5e-2


def test_graph_pdl_and_eager_agree():
    kw = FAMILIES["llama"]
    res = []
    for opts in (dict(), dict(use_cuda_graph=0), dict(use_pdl=1), dict(use_cuda_graph=0, use_pdl=2)):
        spec, eng = make(kw, decode_persistent=0, **opts)
        assert not eng.decode_persistent()
        prompt = synth.prompt_ids(2, 20, spec.vocab)
        eng.begin_infer()
        eng.infer(prompt)
        tok = S.greedy(eng.logits())
        rows = []
        for _ in range(6):
            eng.infer([tok])
            lg = eng.logits()
            rows.append(lg)
            tok = S.greedy(lg)
        res.append(np.stack(rows))
        eng.close()
    for r in res[1:]:
        np.testing.assert_array_equal(res[0], r)


def decode_rows(eng, prompt, steps):
    """Logits of the prefill and of `steps` greedy decode steps."""
    eng.begin_infer()
    eng.infer(prompt)
    lg = eng.logits()
    rows, toks = [lg], []
    for _ in range(steps):
        tok = S.greedy(lg)
        toks.append(tok)
        eng.infer([tok])
        lg = eng.logits()
        rows.append(lg)
    return np.stack(rows), toks


# The persistent GEMV segments compute the projections with the per-op
# kernels' arithmetic order and attention is the same kernel in both paths,
# so the two decode paths agree bit for bit.
@pytest.mark.parametrize("fam", sorted(FAMILIES))
def test_persistent_step_matches_per_op_graph(fam):
    kw = FAMILIES[fam]
    spec, ep = make(kw, decode_persistent=1)
    _, eg = make(kw, decode_persistent=0)
    assert ep.decode_persistent() and not eg.decode_persistent()
    prompt = synth.prompt_ids(5, 40, spec.vocab)
    rp, tp_ = decode_rows(ep, prompt, 16)
    rg, tg = decode_rows(eg, prompt, 16)
    np.testing.assert_array_equal(rp, rg)
    assert tp_ == tg
    ep.close()
    eg.close()


def test_persistent_long_context_and_decode_loop():
    # a context of many attention splits per KV head, then the advance-mode
    # decode loop (graph of cooperative launches) on both paths
    kw = FAMILIES["llama"]
    spec, ep = make(kw, decode_persistent=1)
    _, eg = make(kw, decode_persistent=0)
    prompt = synth.prompt_ids(6, 1500, spec.vocab)
    rp, _ = decode_rows(ep, prompt, 4)
    rg, _ = decode_rows(eg, prompt, 4)
    np.testing.assert_array_equal(rp, rg)
    assert ep.time_decode(8) > 0 and eg.time_decode(8) > 0
    np.testing.assert_array_equal(ep.logits(), eg.logits())
    # timing one segment overwrites the workspace and resets the barrier
    # counters; the following decode steps must be unaffected
    ms, nbytes = ep.time_segment(0, 4)
    assert ms > 0 and nbytes > 0
    tok = S.greedy(eg.logits())
    for _ in range(3):
        ep.infer([tok])
        eg.infer([tok])
        np.testing.assert_array_equal(ep.logits(), eg.logits())
        tok = S.greedy(eg.logits())
    ep.close()
    eg.close()


@pytest.mark.parametrize("fam", sorted(FAMILIES))
def test_prefill_gemm_epilogues_tensor_and_cuda_cores_agree(fam):
    # 300 prompt rows: three 128-row GEMM tiles, the last one partial, through
    # every epilogue (bias, residual add, SwiGLU) of both prefill GEMMs
    spec, et = make(FAMILIES[fam], prefill_tensor_cores=1)
    _, ec = make(FAMILIES[fam], prefill_tensor_cores=0)
    orc = OracleModel(spec, synth.model_weights(spec, 0), mode="f16", kv_gb=2)
    prompt = synth.prompt_ids(7, 300, spec.vocab)
    out = []
    for eng in (et, ec):
        eng.begin_infer()
        st, _ = eng.infer(prompt)
        assert st == E.Status.OK
        out.append(eng.logits())
        eng.close()
    orc.begin_infer()
    _, lo = orc.infer(prompt)
    assert np.max(np.abs(out[0] - out[1])) < LOGIT_TOL
    assert np.max(np.abs(out[0] - lo)) < LOGIT_TOL


def test_kv_capacity_rule_matches_reference():
    z = np.load(os.path.join(GOLDEN, "llama_kvcap.npz"))
    kw = json.loads(str(z["spec"]))
    spec, eng = make(kw, kv_cache_gb=1)
    assert eng.info()["kv_capacity"] == 4096
    eng.begin_infer()
    st, _ = eng.infer(list(z["prompt"]))
    assert st == E.Status.OK
    assert eng.info()["last_kv_index"] == 2047
    st, _ = eng.infer([int(z["ids"][0])])
    assert st == E.Status.OK
    st, _ = eng.infer([int(z["ids"][1])])
    assert st == E.Status.KV_CACHE_EXCEEDED == int(z["error"])
    # reference greedy ids on the FP32 path: FP16 agrees up to near-ties
    lg = eng.logits()
    assert lg.shape == (spec.vocab,)


def test_prompt_of_one_token_stays_in_prefill():
    spec, eng = make(FAMILIES["llama"])
    orc = OracleModel(spec, synth.model_weights(spec, 0), mode="f16")
    eng.begin_infer()
    orc.begin_infer()
    ids = [5]
    for _ in range(4):
        eng.infer(ids)
        _, lo = orc.infer(ids)
        assert eng.info()["last_kv_index"] == 0 == orc.last
        assert np.max(np.abs(eng.logits() - lo)) < LOGIT_TOL
        ids = [S.greedy(lo)]


def test_kv_cache_disabled_and_left_trim():
    kw = dict(model_type="qwen2", max_pos=512)
    spec, eng = make(kw, kv_cache_enabled=0)
    orc = OracleModel(spec, synth.model_weights(spec, 0), mode="f16", kv_enabled=False)
    eng.begin_infer()
    orc.begin_infer()
    ids = list(synth.prompt_ids(0, 508, spec.vocab))
    for step in range(8):
        st, trimmed = eng.infer(ids)
        assert st == E.Status.OK
        _, lo = orc.infer(ids)
        np.testing.assert_array_equal(trimmed, orc.ids)
        assert len(trimmed) <= 512
        assert np.max(np.abs(eng.logits() - lo)) < LOGIT_TOL
        ids = list(trimmed) + [S.greedy(lo)]


def test_infer_before_begin_and_bad_token():
    spec, eng = make(FAMILIES["qwen3"])
    with pytest.raises(E.YlmError) as ei:
        eng.infer([1, 2, 3])
    assert ei.value.status == E.Status.NOT_READY
    eng.begin_infer()
    with pytest.raises(E.YlmError) as ei:
        eng.infer([spec.vocab + 5])
    assert ei.value.status == E.Status.INVALID_ARG
    # the engine stays usable
    eng.begin_infer()
    st, _ = eng.infer([1, 2, 3])
    assert st == E.Status.OK


def test_topk_sampling_bit_exact_against_oracle():
    spec, eng = make(FAMILIES["qwen3"])
    masked = [3, 7, 11, 999]
    seed = 1234
    eng.set_sampling(greedy=False, top_k=40, temperature=0.6, seed=seed, masked_ids=masked)
    eng.begin_infer()
    eng.infer(synth.prompt_ids(3, 16, spec.vocab))
    tok = eng.sample(True)  # the first token is greedy (ChatSession.cpp:140)
    call = 1
    for _ in range(10):
        st, nxt = eng.decode(tok, False)
        assert st == E.Status.OK
        lg = eng.logits(as_float32=True)
        u = sampler_uniform(seed, call)
        want = S.sample_topk(lg, 40, 0.6, u, masked)
        ids, probs, u_used = eng.last_topk()
        assert np.float32(u_used) == u
        vals, want_ids = S.topk_candidates(lg, 40, 0.6, masked)
        np.testing.assert_array_equal(ids, want_ids)
        np.testing.assert_array_equal(probs, S.topk_probs(vals))
        assert nxt == want
        assert nxt not in masked
        tok = nxt
        call += 1


@pytest.mark.parametrize("persistent", [0, 1])
def test_generate_matches_oracle_greedy(persistent):
    spec, eng = make(FAMILIES["llama"], decode_persistent=persistent)
    orc = OracleModel(spec, synth.model_weights(spec, 0), mode="f16")
    prompt = synth.prompt_ids(4, 32, spec.vocab)
    r = eng.generate(prompt, 24, eos_ids=[])
    assert r["status"] == E.Status.OK and len(r["ids"]) == 24
    orc.begin_infer()
    ids = list(prompt)
    for i, t in enumerate(r["ids"]):
        _, lo = orc.infer(ids)
        if S.greedy(lo) != t:
            assert top2_gap(lo) < TIE_GAP
            break
        ids = [int(t)]


def test_llama3_scaled_rope_matches_oracle():
    # rope_scaling = 1: the engine's llama3-scaled table (the reference parses
    # the fields but applies plain theta, so this is checked against the
    # oracle's scaled table, itself pinned to transformers in test_rope_scaling)
    scaling = {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192}
    kw = dict(FAMILIES["llama"], rope_scaling=scaling)
    # weights N(0, 0.06): with N(0, 0.02) the attention of this small model is
    # nearly uniform and the two tables give logits only ~3e-3 apart
    spec, eng = make(kw, rope_scaling=1, init_std=0.06)
    w = synth.model_weights(spec, 0, std=0.06)
    orc = OracleModel(spec, w, mode="f16", rope_scaling=True)
    plain = OracleModel(spec, w, mode="f16", rope_scaling=False)
    prompt = synth.prompt_ids(8, 300, spec.vocab)
    worst, _ = run_teacher_forced(eng, orc, prompt, 8)
    assert worst < LOGIT_TOL
    # the scaled and plain tables give clearly different logits at these positions
    eng.begin_infer()
    plain.begin_infer()
    eng.infer(prompt)
    _, lp = plain.infer(prompt)
    assert np.max(np.abs(eng.logits() - lp)) > 10 * LOGIT_TOL


def test_generate_one_step_behind_stops_and_rolls_back():
    # ylm_generate keeps one decode step in flight; a step launched past an
    # EOS is discarded, so the cache state equals a step-by-step run's
    spec, eng = make(FAMILIES["llama"])
    _, ref = make(FAMILIES["llama"])
    prompt = synth.prompt_ids(12, 32, spec.vocab)
    ids = [int(t) for t in eng.generate(prompt, 20, eos_ids=[])["ids"]]
    assert len(ids) == 20
    stop = next(i for i in range(3, len(ids)) if ids[i] not in ids[:i])
    r = eng.generate(prompt, 20, eos_ids=[ids[stop]])
    assert r["status"] == E.Status.OK
    assert [int(t) for t in r["ids"]] == ids[:stop]
    assert eng.info()["last_kv_index"] == len(prompt) - 1 + stop
    # the same tokens fed one call at a time
    ref.begin_infer()
    ref.infer(prompt)
    for t in ids[:stop + 1]:
        ref.infer([t])
    eng.infer([ids[stop]])
    np.testing.assert_array_equal(eng.logits(), ref.logits())
    # max_new and the greedy ids of the per-token path (kept for a fixed draw)
    r3 = eng.generate(prompt, 7, eos_ids=[])
    assert [int(t) for t in r3["ids"]] == ids[:7]


@pytest.mark.parametrize("layer", [0, 1])
def test_device_wait_times_out_and_engine_recovers(layer):
    # A bounded wait made to run out: the layer's SwiGLU activation goes to a
    # scratch buffer, so the down projection polls words nothing writes.
    # The wait gives up after wait_limit_us, the step's other waits give up at
    # once, the call reports a device timeout, and the next request is exact.
    spec, eng = make(FAMILIES["llama"], wait_limit_us=2000)
    _, ref = make(FAMILIES["llama"])
    assert eng.decode_persistent()
    prompt = synth.prompt_ids(13, 24, spec.vocab)
    eng.begin_infer()
    eng.infer(prompt)
    tok = S.greedy(eng.logits())
    eng.debug_drop_output(layer)
    t0 = time.time()
    with pytest.raises(E.YlmError) as ei:
        eng.infer([tok])
    assert ei.value.status == E.Status.DEVICE_TIMEOUT
    assert time.time() - t0 < 1.0  # the 2 ms bound, not the default 2 s
    eng.debug_drop_output(-1)
    for e in (eng, ref):
        e.begin_infer()
        e.infer(prompt)
    for _ in range(3):
        eng.infer([tok])
        ref.infer([tok])
        np.testing.assert_array_equal(eng.logits(), ref.logits())
        tok = S.greedy(ref.logits())


@pytest.mark.parametrize("fam", ["llama_g8", "qwen2"])
def test_fused_greedy_pick_is_the_argmax(fam):
    # one decode step + greedy sample on the persistent path picks the token in
    # the lm_head epilogue (no sampler launch): the first index of the maximum
    # of the FP16 logits, as torch::argmax and the sampler kernel pick it
    spec, eng = make(FAMILIES[fam])
    assert eng.decode_persistent()
    eng.begin_infer()
    eng.infer(synth.prompt_ids(14, 30, spec.vocab))
    tok = eng.sample(True)
    for _ in range(16):
        st, nxt = eng.decode(tok, True)
        assert st == E.Status.OK
        lg = eng.logits(as_float32=False)
        assert nxt == int(np.argmax(lg))
        tok = nxt


@pytest.mark.parametrize("count", [1, 2, 3])
def test_generate_writes_no_more_than_max_new_ids(count):
    spec, eng = make(FAMILIES["llama"])
    prompt = synth.prompt_ids(12, 32, spec.vocab)
    want = [int(t) for t in eng.generate(prompt, 4, eos_ids=[])["ids"]]
    p = np.asarray(prompt, np.int64)
    out = np.full(16, -77, np.int64)
    n, a, b = ctypes.c_int32(), ctypes.c_double(), ctypes.c_double()
    i64 = ctypes.POINTER(ctypes.c_int64)
    E.check(E.lib().ylm_generate(eng._h, p.ctypes.data_as(i64), p.size, count, None, 0, out.ctypes.data_as(i64),
                                 ctypes.byref(n), ctypes.byref(a), ctypes.byref(b)), "ylm_generate")
    assert n.value == count and out[:count].tolist() == want[:count]
    assert (out[count:] == -77).all()
    # the last slot written belongs to the last step that ran
    assert eng.info()["last_kv_index"] == len(prompt) - 1 + count - 1
