"""CachedDecoder: the decoding operators together, as a generation loop calls
them, between the lowered programs of a small GPT."""
import math

import numpy as np
import pytest

from oracle import decode_ref as R
from oracle.stablehlo_ref import run
from sheaf_b200 import session as S
from sheaf_b200.decode import CachedDecoder
from sheaf_lowering import generate as G
from sheaf_lowering import models as M

from test_decode_ops import U32, attention_bound

C = M.GPTConfig(2, 4, 256, 48, 65, 1, 48)  # heads of 64

# A product of K terms in f32 is off by some K half steps of its result (K half
# steps of the terms' sizes at most, sqrt(K) of them for errors of random sign,
# and a sum of K terms of random sign is sqrt(K) times smaller than its terms):
# two layers of 256 + 256 + 256 + 1024 and the logits' 256.
TOL = (2 * (3 * 256 + 1024) + 256) * U32


def params_of(c, seed):
    """Weights large enough that the logits differ by more than rounding."""
    inp = M.gpt_inputs(c, batch=1, seed=seed)
    return {n: inp[n] * np.float32(1 if inp[n].ndim == 1 else 5) for n, _ in M.gpt_param_leaves(c)}


class HostBuffer:
    def __init__(self, a):
        self.a = a

    shape = property(lambda self: self.a.shape)

    def to_host(self):
        return self.a

    def release(self):
        pass


class OracleSession:
    """The calls that CachedDecoder makes, in numpy: programs by the StableHLO
    oracle, operators by their 64-bit restatement."""

    def __init__(self):
        self.texts, self.largest = {}, 0.0

    def buffer(self, a):
        return HostBuffer(np.array(a))

    def zeros(self, shape, dtype="f32"):
        return HostBuffer(np.zeros(shape, {"f32": np.float32, "i32": np.int32, "int8": np.int8}[dtype]))

    def kv_cache(self, *shape_and_dtype):
        return S.B200Session.kv_cache(self, *shape_and_dtype)

    def has_function(self, name):
        return name in self.texts

    def load_stablehlo(self, text):
        module = text.split("module @", 1)[1].split()[0]
        function = text.split("func.func @", 1)[1].split("(")[0]
        self.texts[f"{module}.{function}"] = text

    def call_device(self, name, args):
        return [HostBuffer(np.array(r)) for r in run(self.texts[name], name, [a.a for a in args])]

    def kv_cache_write(self, cache, at, k, v):
        for c, s, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
            R.write(c.a, None if s is None else s.a, at.a, x.a)

    def kv_cache_attention(self, cache, at, q, out, parents=None):
        kv = [c.a.astype(np.float64) * (1 if s is None else s.a[..., None])
              for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
        out.a[:] = R.attention(*kv, at.a, q.a, 1 / math.sqrt(q.shape[-1]), None if parents is None else parents.a)[0]

    def beam_select(self, logits, scores, out_scores, parents, tokens, finished=None, out_finished=None, eos=-1):
        self.largest = max(self.largest, np.abs(logits.a).max())
        s, p, t, f = R.beam_select(logits.a, scores.a, None if finished is None else finished.a, eos)
        out_scores.a[:], parents.a[:], tokens.a[:] = s, p, t
        if out_finished is not None:
            out_finished.a[:] = f

    def beam_reorder(self, states, parents, axes, lengths=None):
        for st, axis in zip(states, axes):
            st.a[:] = R.reorder(st.a, parents.a, axis, lengths.a)


def full_logits(params, tokens):
    """Logits of every position of one sequence, by the whole forward."""
    c = M.GPTConfig(C.n_layer, C.n_head, C.n_embd, C.block_size, C.vocab_size, 1, len(tokens))
    low = M.gpt_fwd(c, batch=1)
    args = {**params, "idx": np.float32(tokens)[None]}
    return run(low.text, low.qualified, [args[n] for n in low.arg_names])[0][0]


def feed(dec, tokens):
    """tokens [slots, P]: a prompt of two pieces, a token, and a chain; the logits of what they return."""
    n = dec.slots
    dec.prompt(tokens[:, :5], chunk=3)
    one = dec.forward(tokens[:, 5:6], np.full(n, 5)).to_host().reshape(n, 1, -1)
    rest = dec.forward(tokens[:, 6:], np.full(n, 6)).to_host().reshape(n, tokens.shape[1] - 6, -1)
    return np.concatenate([one, rest], 1)


def test_cached_programs_equal_the_full_forward():
    params = params_of(C, 1)
    tokens = np.random.default_rng(2).integers(0, C.vocab_size, (2, 10))
    got = feed(CachedDecoder(OracleSession(), C, params, 2), tokens)
    for n in range(2):
        ref = full_logits(params, tokens[n])[5:]
        assert np.abs(got[n] - ref).max() <= TOL * np.abs(ref).max()


def draft(dec, tokens, tree, parents):
    dec.prompt(tokens)
    n = len(tokens)
    return dec.forward(tree, np.full(n, tokens.shape[1]), parents=parents).to_host().reshape(n, tree.shape[1], -1)


TREE = np.int32([[-1, 0, 0, 1, 2, 4]])


def test_a_tree_gives_the_logits_of_its_paths():
    params = params_of(C, 3)
    rng = np.random.default_rng(4)
    tokens, tree = rng.integers(0, C.vocab_size, (1, 6)), rng.integers(0, C.vocab_size, (1, 6))
    got = draft(CachedDecoder(OracleSession(), C, params, 1), tokens, tree, TREE)
    seen = R.ancestors(TREE[0], 6)
    for t in range(6):
        ref = full_logits(params, np.concatenate([tokens[0], tree[0][seen[t]]]))[-1]
        assert np.abs(got[0, t] - ref).max() <= TOL * np.abs(ref).max()


def plain_beams(params, prompt, W, steps, eos):
    """Beam search of one prompt that keeps whole sequences and reruns the forward."""
    beams = [(0.0, [], False)]
    for _ in range(steps):
        cands = []
        for w, (score, seq, done) in enumerate(beams):
            if done:
                cands.append((score, w, eos, True))
                continue
            z = full_logits(params, list(prompt) + seq)[-1].astype(np.float64)
            lp = z - z.max() - np.log(np.exp(z - z.max()).sum())
            cands += [(score + lp[v], w, v, v == eos) for v in range(len(z))]
        cands.sort(key=lambda x: -x[0])
        beams = [(s, beams[w][1] + [v], d) for s, w, v, d in cands[:W]]
    return beams


def test_beam_search_equals_a_search_without_caches():
    params = params_of(C, 5)
    prompt = np.random.default_rng(6).integers(0, C.vocab_size, (2, 4))
    for eos in (-1, 11):
        sess = OracleSession()
        tokens, scores = CachedDecoder(sess, C, params, 6).beam_search(prompt, 3, 4, eos)
        for g in range(2):
            ref = plain_beams(params, prompt[g], 3, 4, eos)
            assert [list(s) for _, s, _ in ref] == tokens[g].tolist()
            bound = 4 * (2 * TOL * sess.largest + U32 * np.abs(scores[g]))  # two logits enter a score
            assert (np.abs(scores[g] - [s for s, _, _ in ref]) <= bound).all()


def test_calls_that_do_not_fit_are_refused():
    dec = CachedDecoder(OracleSession(), C, params_of(C, 1), 2)
    one = np.zeros((2, 1))
    for call in (lambda: dec.forward(np.zeros((3, 1)), [0, 0]), lambda: dec.forward(one, [0, C.block_size]),
                 lambda: dec.forward(one, [0]), lambda: dec.forward(one, [0, 0], parents=[[0], [0], [0]]),
                 lambda: dec.forward(np.zeros((2, 0)), [0, 0]), lambda: dec.beam_search(one, 2, 3),
                 lambda: dec.beam_search(one[:1], 2, C.block_size + 1), lambda: dec.beam_search(one[:1], 2, 0)):
        with pytest.raises(S.B200Error) as e:
            call()
        assert e.value.code == 3


# ------------------------------------------------------------------ device

class CheckedSession:
    """A device session whose every operator call is compared with its 64-bit
    restatement, on the very buffers of the call."""

    def __init__(self, sess, kind):
        self.s, self.kind, self.calls = sess, kind, 0

    def __getattr__(self, name):
        return getattr(self.s, name)

    def arrays(self, cache):
        return [(c.to_host().copy(), s if s is None else s.to_host().copy())
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]

    def kv_cache_write(self, cache, at, k, v):
        want = self.arrays(cache)
        self.s.kv_cache_write(cache, at, k, v)
        for (a, s), (got, gs), x in zip(want, self.arrays(cache), (k, v)):
            R.write(a, s if self.kind == "int8" else self.kind, at.to_host(), x.to_host())
            assert np.array_equal(a, got) and (s is None or np.array_equal(s, gs))
        self.calls += 1

    def kv_cache_attention(self, cache, at, q, out, parents=None):
        self.s.kv_cache_attention(cache, at, q, out, parents=parents)
        k, v = (a.astype(np.float64) * (1 if s is None else s.astype(np.float64)[..., None])
                for a, s in self.arrays(cache))
        D = q.shape[-1]
        ref, dots, vmax, live = R.attention(k, v, at.to_host(), q.to_host(), np.float32(1 / math.sqrt(D)),
                                            None if parents is None else parents.to_host())
        assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, "f32")).all()
        self.calls += 1

    def beam_reorder(self, states, parents, axes, lengths=None):
        old = [s.to_host().copy() for s in states]
        self.s.beam_reorder(states, parents, axes, lengths=lengths)
        for a, st, axis in zip(old, states, axes):
            assert np.array_equal(R.reorder(a, parents.to_host(), axis, lengths.to_host()), st.to_host())
        self.calls += 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "int8"])
def test_device_decoder_call_by_call(fp32_session, kind):
    """Prompt, single tokens, a chain, a tree and a beam search; with f32 caches
    the logits and the beams are those of the oracle session's."""
    params = params_of(C, 7)
    rng = np.random.default_rng(8)
    tokens, tree = rng.integers(0, C.vocab_size, (2, 10)), rng.integers(0, C.vocab_size, (2, 6))
    parents = np.repeat(TREE, 2, axis=0)
    prompt = rng.integers(0, C.vocab_size, (2, 4))

    def decoder(sess, slots):
        return CachedDecoder(sess, C, params, slots, kind)
    checked = CheckedSession(fp32_session, kind)
    got = [feed(decoder(checked, 2), tokens), draft(decoder(checked, 2), tokens, tree, parents)]
    beams = [decoder(checked, 6).beam_search(prompt, 3, 4, eos) for eos in (-1, 11)]
    assert checked.calls > 0
    if kind != "f32":
        return
    sess = OracleSession()
    want = [feed(decoder(sess, 2), tokens), draft(decoder(sess, 2), tokens, tree, parents)]
    for a, b in zip(got, want):
        assert np.abs(a - b).max() <= TOL * np.abs(b).max()
    for (tok, score), eos in zip(beams, (-1, 11)):
        rt, rs = decoder(sess, 6).beam_search(prompt, 3, 4, eos)
        assert np.array_equal(tok, rt)
        assert (np.abs(score - rs) <= 4 * (2 * TOL * sess.largest + U32 * np.abs(rs) + 2.4e-6)).all()


@pytest.mark.gpu
def test_device_idle_slots_and_refusals(fp32_session):
    """A slot with a negative position neither changes its caches nor the other's logits."""
    params = params_of(C, 9)
    tokens = np.random.default_rng(10).integers(0, C.vocab_size, (2, 3))
    dec = CachedDecoder(fp32_session, C, params, 2, "int8")
    both = dec.forward(tokens, [0, 0]).to_host()
    before = [b.to_host() for c in dec.caches for b in c.buffers()]
    alone = dec.forward(tokens, [0, -1]).to_host()
    assert np.array_equal(both[:3], alone[:3])
    for a, b in zip(before, (b.to_host() for c in dec.caches for b in c.buffers())):
        assert np.array_equal(a, b)
    with pytest.raises(S.B200Error):
        dec.forward(np.zeros((2, 65)), [0, 0])


def test_positions_near_the_ends_of_their_type():
    """Positions whose end passes 32 bits are refused; far negative ones are idle slots."""
    dec = CachedDecoder(OracleSession(), C, params_of(C, 1), 2)
    for far in (2 ** 31 - 1, 2 ** 31, 2 ** 40):
        with pytest.raises(S.B200Error) as e:
            dec.forward(np.zeros((2, 1)), [0, far])
        assert e.value.code == 3
    idle = [dec.forward(np.zeros((2, 1)), [0, far]).to_host() for far in (-1, -2 ** 31, -2 ** 40)]
    assert np.array_equal(idle[0][0], idle[1][0]) and np.array_equal(idle[0][0], idle[2][0])
