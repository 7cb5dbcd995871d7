"""The decoding operators (key/value cache write, read and attention; beam
selection and reordering) against the 64-bit restatement in
oracle/decode_ref.py, through the C ABI."""
import ctypes
import math

import numpy as np
import pytest

from oracle import decode_ref as R
from sheaf_b200 import session as S

U32 = 2.0 ** -24   # half a step of f32, relative
UBF = 2.0 ** -8    # half a step of bf16, relative
KINDS = ("f32", "bf16", "int8")


# ------------------------------------------------------------------ host (no GPU)

def test_oracle_codes_round_ties_to_even_and_keep_the_largest():
    x = np.float32([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -127.0]])
    q, s = R.quantise(x)
    assert s[0] == 1.0 and q.tolist() == [[127, 0, 2, 2, 0, -2, 126, -127]]
    q, s = R.quantise(np.zeros((1, 4), np.float32))
    assert s[0] == 0 and not q.any()


def test_oracle_ancestors_of_a_tree_and_a_chain():
    seen = R.ancestors([-1, 0, 0, 1, 9, -7], 6)
    assert [np.flatnonzero(r).tolist() for r in seen] == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [5]]
    assert (R.ancestors(None, 5) == np.tril(np.ones((5, 5), bool))).all()


def test_oracle_beam_first_step_and_finished_beams():
    logits = np.log(np.float64([[0.5, 0.3, 0.2]] * 2))
    s, p, t, f = R.beam_select(logits, np.float32([[0, -np.inf]]))
    assert p.tolist() == [[0, 0]] and t.tolist() == [[0, 1]]
    s, p, t, f = R.beam_select(logits, np.float32([[-1, -0.1]]), np.int32([[0, 1]]), 2)
    assert p.tolist() == [[1, 0]] and t.tolist() == [[2, 0]] and f.tolist() == [[1, 0]]


def test_oracle_reorder_reads_the_old_rows():
    x = np.arange(8, dtype=np.float32).reshape(4, 2)
    got = R.reorder(x, np.int32([[1, 0], [1, 5]]), 1, np.int32([1, 2, 0, 1]))
    assert got.tolist() == [[2, 3], [0, 3], [6, 5], [6, 7]]


def test_null_arguments_are_refused_on_the_host(lib):
    cache = S._KvCache()
    calls = [lib.sb_kv_cache_write(None, cache, None, None, None),
             lib.sb_kv_cache_read(None, cache, None, None, None, None),
             lib.sb_kv_cache_attention(None, cache, None, None, None, 1.0, None),
             lib.sb_beam_select(None, None, None, None, -1, None, None, None, None),
             lib.sb_beam_reorder(None, 0, None, None, None, None),
             lib.sb_buffer_allocate_zero(None, 0, None, S.ELEMENT_TYPE_INT_8, None)]
    for st in calls:
        assert st and lib.sb_status_code_of(st) == 3
        lib.sb_status_free(st)


def test_python_checks_before_the_library():
    s = object.__new__(S.B200Session)
    with pytest.raises(S.B200Error):
        s.kv_cache(1, 1, 8, 16, dtype="int4")
    with pytest.raises(S.B200Error):
        s.beam_reorder([None], None, [1, 2])


# ------------------------------------------------------------------ device

@pytest.fixture(scope="module")
def sess(lib):
    s = S.B200Session(device=0, precision="fp32")
    yield s
    s.close()


def put(sess, a, kind=None):
    """Device copy of a host array; bf16 arrays hold bf16 values as f32."""
    a = np.ascontiguousarray(a)
    if kind == "bf16":
        return sess.buffer(a, bf16=True)
    if a.dtype == np.int8:
        import torch
        b = sess.wrap_torch(torch.from_numpy(a).cuda())
        torch.cuda.synchronize()
        return b
    return sess.buffer(a)


def rand(rng, shape, kind="f32"):
    x = rng.standard_normal(shape).astype(np.float32)
    return R.bf16_round(x) if kind == "bf16" else x


def make_cache(sess, rng, shape, kind, fill=None):
    """A filled device cache, its arrays (values or codes) and its scales."""
    arrays, scales = [], []
    for _ in range(2):
        if kind == "int8":
            arrays.append(rng.integers(-127, 128, shape).astype(np.int8))
            scales.append((rng.random(shape[:3]) * 0.02 + 0.005).astype(np.float32))
        else:
            arrays.append(rand(rng, shape, kind) if fill is None else np.full(shape, fill, np.float32))
    bufs = [put(sess, a, kind) for a in arrays] + [put(sess, s) for s in scales]
    return S.KVCache(*bufs), arrays, scales


def values(arrays, scales):
    if not scales:
        return [a.astype(np.float64) for a in arrays]
    return [a.astype(np.float64) * s.astype(np.float64)[..., None] for a, s in zip(arrays, scales)]


WRITE_SHAPES = [  # slots, tokens, heads, capacity, head size
    (1, 1, 1, 1, 16), (1, 1, 6, 16, 64), (3, 5, 2, 9, 48), (2, 7, 3, 12, 80), (5, 2, 1, 4, 256), (2, 33, 4, 40, 128),
    (4, 3, 5, 8, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", WRITE_SHAPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_write_then_read(sess, shape, kind, src):
    N, n_tok, H, T, D = shape
    rng = np.random.default_rng([*shape, KINDS.index(kind), len(src)])
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    pos = rng.integers(0, max(1, T - n_tok + 1), N).astype(np.int32)
    if N > 1:
        pos[0] = -1 if N > 2 else T - 1          # idle, or running over the capacity
        pos[-1] = 2 ** 31 - 1 if N > 3 else T - 1
    x = [rand(rng, (N, n_tok, H, D), src) for _ in range(2)]
    sess.kv_cache_write(cache, put(sess, pos), put(sess, x[0], src), put(sess, x[1], src))
    want = [a.copy() for a in arrays]
    wscale = [s.copy() for s in scales]
    for i in range(2):
        R.write(want[i], wscale[i] if kind == "int8" else kind, pos, x[i])
    got = cache.buffers()
    for i in range(2):
        assert np.array_equal(got[i].to_host(), want[i])
        if kind == "int8":
            assert np.array_equal(got[2 + i].to_host(), wscale[i])
    # read back: a window that starts before and ends after the cache, ragged counts
    rows = T + 3
    starts = rng.integers(-2, T + 1, N).astype(np.int32)
    counts = rng.integers(-1, rows + 2, N).astype(np.int32)
    for out in ("f32", "bf16"):
        before = [rand(rng, (N, H, rows, D), out) for _ in range(2)]
        outs = [put(sess, b, out) for b in before]
        sess.kv_cache_read(cache, outs[0], outs[1], starts=put(sess, starts), counts=put(sess, counts))
        for i in range(2):
            ref = before[i].copy()
            val = want[i] if kind != "int8" else want[i].astype(np.float32) * wscale[i][..., None]
            for n in range(N):
                for r in range(min(rows, max(0, int(counts[n])))):
                    t = int(starts[n]) + r
                    if 0 <= t < T:
                        ref[n, :, r] = R.bf16_round(val[n, :, t]) if out == "bf16" else val[n, :, t]
            assert np.array_equal(outs[i].to_host(), ref)
    # the whole cache, no starts and counts
    outs = [sess.zeros((N, H, T, D)) for _ in range(2)]
    sess.kv_cache_read(cache, outs[0], outs[1])
    for i in range(2):
        val = want[i] if kind != "int8" else want[i].astype(np.float32) * wscale[i][..., None]
        assert np.array_equal(outs[i].to_host(), val)


@pytest.mark.gpu
def test_write_codes_of_hard_rows(sess):
    """Ties, zeros, subnormal rows, NaN and infinities: codes and scales are the
    definition's, exactly."""
    rng = np.random.default_rng(5)
    D, rows = 64, []
    rows.append(np.zeros(D))
    rows.append(np.r_[127.0, np.arange(63) - 31.5])                     # ties at scale 1
    rows.append(np.r_[127.0, np.arange(63) - 31.5] * 2.0 ** -130)      # the same with a subnormal scale
    rows.append(np.full(D, 2.0 ** -149))                               # the scale rounds to 0
    rows.append(np.r_[190 * 2.0 ** -149, np.full(63, 2.0 ** -149)])     # scale one step, code clamped
    rows.append(np.r_[np.nan, np.inf, -np.inf, rng.standard_normal(61)])
    rows.append(np.r_[3.4028234e38, rng.standard_normal(63) * 1e37])
    s = np.float32(0.1237)
    k = np.arange(63) - 31
    rows.append(np.r_[np.float32(127 * s), (k + 0.5) * s])               # next to ties of a scale that is not a power of 2
    x = np.float32(rows + [np.float32(rng.standard_normal(D) * 10.0 ** e) for e in range(-40, 39)])
    x = x.reshape(1, len(x), 1, D)
    cache = sess.kv_cache(1, 1, x.shape[1], D, "int8")
    zero = put(sess, np.int32([0]))
    sess.kv_cache_write(cache, zero, put(sess, x), put(sess, -x))
    for b, sc, y in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, -x)):
        q, s = R.quantise(y[0, :, 0])
        assert np.array_equal(sc.to_host()[0, 0], s)
        assert np.array_equal(b.to_host()[0, 0], q)


def attention_bound(dots, vmax, live, D, out, kind):
    """How far an f32 evaluation may be from the 64-bit result, per element.
    A score is D products added in f32 with q pre-scaled: at most (D + 4) half
    steps of sum |q k| scale, in units of log2 e less than 2 of it; a relative
    error of e in every probability moves the output by at most 2 e max|v|;
    exp2 and the running rescalings add a few half steps per term and the sums
    at most one per addition (`live` of them).  A bf16 evaluation may also round
    each probability (times its value row's scale) to bf16 before the second
    product: each term p v moves by at most half a bf16 step of itself, so the
    output by at most UBF sum p |v| <= UBF max|v|; and it rounds the output."""
    e = 2 * (D + 4) * U32 * dots + (live + 64) * U32
    b = 2 * e * vmax
    if kind == "bf16":
        b = b + UBF * vmax + UBF * np.abs(out).max(-1)
    return b[..., None]


ATT_CASES = [  # slots, tokens, q heads, heads, capacity, head size, positions
    (1, 1, 1, 1, 1, 16, [0]),
    (1, 1, 6, 6, 256, 64, [200]),
    (4, 1, 4, 4, 70, 64, [-1, 0, 69, 70]),            # idle, first token, last place, full
    (3, 1, 8, 2, 133, 128, [1, 64, 132]),
    (2, 1, 6, 2, 40, 80, [7, 39]),
    (2, 1, 2, 2, 37, 256, [36, 2 ** 31 - 1]),
    (2, 1, 5, 1, 90, 32, [17, 88]),
    (2, 5, 3, 3, 50, 48, [0, 44]),
    (3, 7, 4, 2, 60, 64, [3, 56, -5]),                # the tokens run over the capacity; idle
    (1, 64, 2, 2, 300, 64, [200]),
    (2, 63, 8, 4, 130, 128, [0, 66]),
    (1, 64, 16, 2, 200, 128, [130]),
    (2, 16, 4, 4, 1100, 64, [1000, 513]),
    (1, 33, 8, 1, 777, 64, [700]),
    (1, 9, 4, 2, 70, 256, [50]),
    (2, 12, 2, 1, 33, 16, [20, 30]),
    (2, 10, 6, 3, 75, 48, [20, 70]),
    (1, 20, 4, 2, 140, 96, [100]),
    (2, 8, 4, 2, 150, 112, [9, 140]),
    (1, 64, 3, 1, 200, 64, [130]),                    # 192 rows
    (2, 3, 4, 2, 300, 64, [250, 30]),
    (1, 8, 2, 2, 500, 128, [450]),
    (2, 5, 2, 2, 90, 32, [80, 87]),
]


def tree_of(rng, N, n_tok):
    p = np.zeros((N, n_tok), np.int32)
    for n in range(N):
        for s in range(n_tok):
            p[n, s] = rng.integers(max(-1, s - 6), s) if s else -1
    if n_tok > 4:  # values outside [0, t) end the path
        p[0, 3], p[-1, 4] = 3, -9
        p[0, n_tok - 1] = 2 ** 31 - 1
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("case,tree", [(c, t) for c in ATT_CASES for t in (False, True) if c[1] > 1 or not t],
                         ids=lambda c: "x".join(map(str, c[:6])) if isinstance(c, tuple) else "tree" if c else "chain")
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_attention(sess, case, kind, src, tree):
    N, n_tok, Hq, H, T, D, pos = case
    rng = np.random.default_rng(n_tok * 1000 + T + D)
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    q = rand(rng, (N, n_tok, Hq, D), src)
    parents = tree_of(rng, N, n_tok) if tree else None
    scale = 1 / math.sqrt(D) if not tree else 0.3
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, scale, parents)
    out = put(sess, np.full(q.shape, 7.0, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out,
                            parents=None if parents is None else put(sess, parents), scale=None if not tree else scale)
    got = out.to_host()
    assert (np.abs(got - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()
    assert not got[live == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D,T", [(1, 1, 64, 9000), (1, 4, 128, 5000), (3, 4, 64, 6000), (1, 1, 256, 3000),
                                         (1, 2, 32, 4000)])
def test_attention_of_one_long_sequence(sess, kind, src, n_tok, G, D, T):
    """Few (slot, head) pairs over many keys: the widest splits; the second slot leaves most of them empty."""
    N, H = 2, 2
    rng = np.random.default_rng(T + D)
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    q = rand(rng, (N, n_tok, G * H, D), src)
    pos = [T - n_tok - 1, 70]
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, 1 / math.sqrt(D))
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("N,H,n_tok", [(71, 8, 1), (128, 4, 2), (131, 4, 1)])
def test_attention_of_many_uneven_slots(sess, kind, src, N, H, n_tok):
    """More (slot, head) pairs than run at once; idle, empty, equal and full slots among them."""
    T, D = 150, 64
    rng = np.random.default_rng(N)
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    pos = rng.integers(0, T, N)
    pos[[0, 5, 9, 30]] = -1, 0, 2 ** 31 - 1, -7
    pos[40:50] = 77
    q = rand(rng, (N, n_tok, H, D), src)
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, 1 / math.sqrt(D))
    out = put(sess, np.full(q.shape, 7.0, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 40.0])
@pytest.mark.parametrize("n_tok,G,D", [(1, 2, 64), (20, 2, 64), (40, 4, 128)])
def test_attention_scales(sess, kind, src, scale, n_tok, G, D):
    """Scales of 0, negative, and large enough that maxima move by far more than
    an exponent range between tiles."""
    rng = np.random.default_rng(n_tok)
    N, H, T, pos = 1, 2, 700, [600]
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    if not scales:  # growing keys: later tiles hold larger scores
        for a in arrays:
            a *= np.linspace(0.1, 1, T, dtype=np.float32)[:, None]
            a[...] = R.bf16_round(a)
        cache = S.KVCache(*[put(sess, a, kind) for a in arrays])
    q = rand(rng, (N, n_tok, G * H, D), src)
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, scale)
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out, scale=scale)
    assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", [(1, 1, 64), (1, 4, 128), (6, 2, 64), (20, 2, 64), (12, 1, 32)])
@pytest.mark.parametrize("e", [-110, 115])
def test_attention_of_ordinary_scores_from_extreme_factors(sess, src, n_tok, G, D, e):
    """Queries near an end of f32's range over int8 keys whose scales undo it (both by powers of two)."""
    rng = np.random.default_rng(n_tok + D)
    N, H, T = 2, 2, 90
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), "int8")
    scales[0] = np.ldexp(scales[0], -e)
    cache.k_scale = put(sess, scales[0])
    q = np.ldexp(rand(rng, (N, n_tok, G * H, D), src), e)
    pos = [T - n_tok, 17]
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, 1 / math.sqrt(D))
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", [(1, 1, 64), (1, 4, 128), (6, 2, 64), (40, 2, 64), (40, 4, 128)])
def test_attention_ignores_what_it_does_not_attend_to(sess, kind, src, n_tok, G, D):
    """NaN and infinities behind the last token, and in drafted tokens that are
    no ancestors, change nothing; a NaN in an ancestor reaches its descendants."""
    rng = np.random.default_rng(n_tok + G)
    N, H, T, pos = 2, 2, 210, [150, 33]
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    q = rand(rng, (N, n_tok, G * H, D), src)
    parents = np.full((N, n_tok), -1, np.int32)
    if n_tok > 5:
        parents[:, 5] = 2
    run = lambda: _attend(sess, arrays, scales, kind, pos, q, src, parents)
    clean = run()
    bad = [np.nan, np.inf, -np.inf]
    for n in range(N):
        for t in range(pos[n] + n_tok, T):
            for i in range(2):
                if scales:
                    scales[i][n, :, t] = bad[t % 3]
                else:
                    arrays[i][n, :, t] = bad[t % 3]
    assert np.array_equal(run(), clean)
    if n_tok > 5:
        for n in range(N):
            for i in range(2):
                if scales:
                    scales[i][n, :, pos[n] + 2] = np.nan
                else:
                    arrays[i][n, :, pos[n] + 2] = np.nan
        got = run()
        others = [s for s in range(n_tok) if s not in (2, 5)]
        assert np.isnan(got[:, [2, 5]]).all()
        # a kernel may treat tokens next to bad values in another order of operations: the probabilities' rounding
        # and the output's, each at most half a step of the output's type on either side, times the largest value
        vmax = max(np.abs(values(arrays, scales)[1][n, :, :pos[n] + 2]).max() for n in range(N))
        step = UBF if src == "bf16" else 2.0 ** -17
        assert (np.abs(got[:, others] - clean[:, others]) <= 4 * step * vmax).all()


def _attend(sess, arrays, scales, kind, pos, q, src, parents):
    cache = S.KVCache(*([put(sess, a, kind) for a in arrays] + [put(sess, s) for s in scales]))
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out, parents=put(sess, parents))
    return out.to_host()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_attention_over_a_cache_beyond_32_bit_offsets(sess, kind, src):
    """2^31 values and more per buffer: the last slot's rows are found."""
    import torch
    N, H, T, D = 3, 1, 6_000_000, 128
    free = torch.cuda.mem_get_info()[0]
    if free < 16 << 30:
        pytest.skip("not enough memory")
    rng = np.random.default_rng(11)
    cache = sess.kv_cache(N, H, T, D, kind)
    pos = np.int32([5, T - 2, T - 1])
    n_tok = 2
    x = [rand(rng, (N, n_tok, H, D)) for _ in range(2)]
    sess.kv_cache_write(cache, put(sess, pos), put(sess, x[0]), put(sess, x[1]))
    outs = [sess.zeros((N, H, n_tok, D)) for _ in range(2)]
    sess.kv_cache_read(cache, outs[0], outs[1], starts=put(sess, pos))
    vals = [o.to_host().astype(np.float64) for o in outs]
    for i in range(2):
        q, s = R.quantise(x[i])
        want = q.astype(np.float32) * s[..., None] if kind == "int8" else R.bf16_round(x[i])
        for n in range(N):
            for t in range(n_tok):
                if pos[n] + t < T:
                    assert np.array_equal(vals[i][n, :, t].astype(np.float32), want[n, t])
    # every other key is zero: its score is 0, its value 0
    qv = rand(rng, (N, n_tok, 1, D), src) * 4
    qv = R.bf16_round(qv)
    out = put(sess, np.zeros(qv.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, pos), put(sess, qv, src), out, scale=0.25)
    got = out.to_host()
    for n in range(N):
        for s in range(n_tok):
            e = [(np.exp(0.25 * float(vals[0][n, 0, j] @ qv[n, s, 0])), vals[1][n, 0, j]) for j in range(s + 1)
                 if pos[n] + j < T]
            total = min(int(pos[n]), T) + sum(a for a, _ in e)
            ref = sum(a * b for a, b in e) / total
            # sums of 6e6 equal terms: each lane adds a fraction of them in order
            tol = (2 * 132 * U32 * 100 + T / 256 * U32) * np.abs(ref).max() + (UBF * np.abs(ref).max() if src == "bf16" else 0)
            assert np.abs(got[n, s, 0] - ref).max() <= tol + 1e-12
    cache.release()


SELECT_CASES = [  # groups, beams, vocabulary
    (1, 1, 1), (1, 1, 2), (1, 4, 65), (3, 5, 7), (2, 16, 3), (2, 16, 16), (4, 8, 1000), (1, 16, 50257), (2, 3, 4097),
    (70, 2, 129), (1, 7, 131071), (5, 8, 50304)]


@pytest.mark.gpu
@pytest.mark.parametrize("G,W,V", SELECT_CASES)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("ends", [False, True])
def test_beam_select(sess, G, W, V, kind, ends):
    rng = np.random.default_rng(G + 10 * W + V)
    logits = (rng.standard_normal((G * W, V)) * 3).astype(np.float32)
    if kind == "bf16":
        logits = R.bf16_round(logits)  # many equal logits
    scores = -np.sort(rng.random((G, W)) * 9).astype(np.float32)
    eos = V // 2 if ends else -1
    fin = (rng.random((G, W)) < 0.4).astype(np.int32)
    check_select(sess, logits, scores, fin, eos, kind)


def check_select(sess, logits, scores, fin, eos, kind="f32"):
    ref = R.beam_select(logits, scores, fin, eos)
    sc, fi = put(sess, scores), put(sess, fin)
    par, tok = sess.zeros(scores.shape, "i32"), sess.zeros(scores.shape, "i32")
    # scores and flags in place, as a search loop keeps them
    if eos >= 0:
        sess.beam_select(put(sess, logits, kind), sc, sc, par, tok, finished=fi, out_finished=fi, eos=eos)
        assert np.array_equal(fi.to_host(), ref[3])
    else:
        sess.beam_select(put(sess, logits, kind), sc, sc, par, tok)
    assert np.array_equal(par.to_host(), ref[1])
    assert np.array_equal(tok.to_host(), ref[2])
    # The sums of f32 exponentials: a term 2^-t is off by 2^-22 (exp2) + 2^-23.4 t
    # of itself (its argument's two roundings); t weighted by 2^-t averages at
    # most log2(V) < 17 here; a term passes at most 9 f32 additions:
    # 2^-22 + 17 * 2^-23.4 + 9 * 2^-24 < 2.4e-6, and the value is rounded once.
    got = sc.to_host().astype(np.float64)
    same = got == ref[0]
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(got - ref[0]) <= U32 * np.abs(ref[0]) + 2.4e-6)).all()


@pytest.mark.gpu
def test_beam_select_ties_masks_and_bad_values(sess):
    rng = np.random.default_rng(2)
    W, V = 6, 3000
    zero = np.zeros((1, W), np.int32)
    # every logit equal: the lowest tokens of the best beam, and of equal beams in turn
    check_select(sess, np.zeros((W, V), np.float32), np.float32([[-1] * W]), zero, -1)
    check_select(sess, np.zeros((W, V), np.float32), np.float32([[0] + [-np.inf] * (W - 1)]), zero, 7)
    # identical beams (same prefix): exact ties between beams
    row = rng.standard_normal((1, V)).astype(np.float32)
    check_select(sess, np.repeat(row, W, 0), np.float32([[-2] * W]), zero, -1)
    # all but a few tokens masked, a whole beam masked, NaN, the lowest finite value, infinities
    x = np.full((W, V), -np.inf, np.float32)
    x[0, [5, 2999]] = [1.0, 1.0]
    x[1, 17] = -3e38
    x[2] = np.finfo(np.float32).min
    x[3] = np.nan
    x[4, 3] = np.inf
    check_select(sess, x, np.float32([[-1, -2, -3, -4, -5, -6]]), zero, -1)
    check_select(sess, x, np.float32([[-np.inf, np.nan, -3, -4, -5, np.inf]]), zero, 2)
    # every beam finished
    check_select(sess, rng.standard_normal((W, V)).astype(np.float32), -np.float32([[1, 5, 2, 2, 9, 0]]), zero + 1, 0)
    # values that differ beyond 32 bits only: the sums decide between beams
    base = rng.standard_normal(V).astype(np.float32)
    x = np.stack([base] * W)
    x[1:, -1] += np.float32([1e-3, 2e-3, 3e-3, 4e-3, 5e-3])
    check_select(sess, x, np.float32([[-40] * W]), zero, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("G,W", [(1, 1), (1, 2), (3, 3), (2, 8), (1, 16), (5, 11)])
def test_beam_reorder(sess, G, W):
    rng = np.random.default_rng(W)
    N = G * W
    T = 19
    states = [(rand(rng, (N, 3, T, 16)), 2, None), (rand(rng, (N, 2, T, 48), "bf16"), 2, "bf16"),
              (rng.integers(-127, 128, (N, 2, T, 16)).astype(np.int8), 2, None), (rand(rng, (N, 3, T)), 2, None),
              (rng.integers(0, 99, (N, T)).astype(np.int32), 1, None), (rand(rng, (N, 5), "bf16"), -1, "bf16"),
              (rng.integers(-9, 9, (N, 7)).astype(np.int8), 1, None), (rand(rng, (N,)), -1, None),
              (rand(rng, (N, T, 3, 2)), 1, None), (rand(rng, (N, 2, 0, 4)), 2, None)]
    states += [(rng.integers(0, 9, (N, 2)).astype(np.int32), -1, None) for _ in range(50)]  # two launches
    parents = rng.integers(0, W, (G, W)).astype(np.int32)
    if W > 2:
        parents[0, 1], parents[-1, 2] = W, -1  # out of range: the row stays
    lengths = rng.integers(-1, T + 3, N).astype(np.int32)
    for lens in (None, lengths):
        bufs = [put(sess, a, k) for a, _, k in states]
        sess.beam_reorder(bufs, put(sess, parents), [ax for _, ax, _ in states],
                          lengths=None if lens is None else put(sess, lens))
        for b, (a, ax, _) in zip(bufs, states):
            assert np.array_equal(b.to_host(), R.reorder(a, parents, ax, lens)), (a.shape, ax)


@pytest.mark.gpu
def test_refusals_launch_nothing(sess, lib):
    import torch
    other = S.B200Session(device=0, precision="fp32")
    z = sess.zeros
    c8, c32 = sess.kv_cache(2, 2, 8, 32, "int8"), sess.kv_cache(2, 2, 8, 32)
    pos = z((2,), "i32")
    kv = [z((2, 1, 2, 32)) for _ in range(2)]
    q, out = z((2, 1, 4, 32)), z((2, 1, 4, 32))
    n0 = lib.sb_kernel_launch_count()

    def refused(f, *a, **k):
        with pytest.raises(S.B200Error) as e:
            f(*a, **k)
        assert e.value.code == 3

    w = lambda c, p=pos, k=kv[0], v=kv[1]: sess.kv_cache_write(c, p, k, v)
    refused(w, S.KVCache(c8.k, c8.v))                                   # int8 without scales
    refused(w, S.KVCache(c32.k, c32.v, c8.k_scale, c8.v_scale))         # f32 with scales
    refused(w, S.KVCache(c32.k, c8.v, c8.k_scale, c8.v_scale))          # types differ
    refused(w, S.KVCache(c32.k, c32.k))                                 # one buffer for both
    refused(w, S.KVCache(c8.k, c8.v, c8.k_scale, z((2, 2, 9))))         # scale shape
    refused(w, S.KVCache(None, c32.v))
    for d in (8, 24, 272):
        refused(w, sess.kv_cache(2, 2, 8, d), k=z((2, 1, 2, d)), v=z((2, 1, 2, d)))
    refused(w, c32, p=z((3,), "i32"))
    refused(w, c32, p=z((2,)))                                          # positions are i32
    refused(w, c32, p=other.zeros((2,), "i32"))                         # another session's buffer
    refused(w, c32, k=z((2, 1, 2, 16)))
    refused(w, c32, k=z((2, 1, 32)))
    refused(w, c32, k=z((2, 1, 2, 32), "bf16"))                         # k and v differ
    refused(w, c32, k=None)
    refused(sess.kv_cache_read, c32, z((2, 2, 4, 32)), z((2, 2, 5, 32)))
    refused(sess.kv_cache_read, c32, z((2, 2, 4, 32), "i32"), z((2, 2, 4, 32), "i32"))
    refused(sess.kv_cache_read, c32, c32.k, z((2, 2, 8, 32)))           # out of the cache into itself
    refused(sess.kv_cache_read, c32, z((2, 2, 4, 32)), z((2, 2, 4, 32)), starts=z((1,), "i32"))
    off = sess.wrap_torch(torch.zeros(2 * 2 * 8 * 32 + 4, device="cuda")[4:].view(2, 2, 8, 32))
    refused(w, S.KVCache(off, c32.v))                                   # 16-byte aligned f32 rows
    a = sess.kv_cache_attention
    refused(a, c32, pos, q, q)
    refused(a, c32, pos, z((2, 1, 3, 32)), z((2, 1, 3, 32)))            # 3 query heads on 2
    refused(a, c32, pos, z((2, 65, 2, 32)), z((2, 65, 2, 32)))          # more than 64 tokens
    refused(a, c32, pos, q, z((2, 1, 4, 32), "bf16"))
    refused(a, c32, pos, q, out, parents=z((2, 2), "i32"))
    refused(a, c32, pos, q, out, scale=float("nan"))
    refused(a, c32, None, q, out)
    lg, sc, i1, i2, i3 = z((4, 9)), z((2, 2)), z((2, 2), "i32"), z((2, 2), "i32"), z((2, 2), "i32")
    b = sess.beam_select
    refused(b, lg, z((2, 3)), z((2, 3)), i1, i2)
    refused(b, z((34, 9)), z((2, 17)), z((2, 17)), z((2, 17), "i32"), z((2, 17), "i32"))
    refused(b, z((4, 0)), sc, sc, i1, i2)
    refused(b, lg, sc, sc, i1, i1)
    refused(b, lg, sc, sc, i1, i2, eos=3)                               # an end token needs the flags
    refused(b, lg, sc, sc, i1, i2, finished=i3, out_finished=i3, eos=9)
    refused(b, lg, sc, sc, i1, i2, finished=i3, out_finished=i3)
    refused(b, lg, sc, sc, i1, i2, finished=i1, out_finished=i3, eos=1)
    refused(b, z((4, 9), "i32"), sc, sc, i1, i2)
    par = z((2, 2), "i32")
    r = sess.beam_reorder
    refused(r, [z((3, 4))], par, [1])
    refused(r, [z((4, 4))], par, [2])
    refused(r, [z((4, 4))], par, [0])
    refused(r, [z((4, 4))], z((4,), "i32"), [1])
    refused(r, [lg, lg], par, [1, 1])
    refused(r, [z((4, 4))], par, [1], lengths=z((2,), "i32"))
    refused(r, [None], par, [1])
    lens = z((4,), "i32")
    refused(r, [lens], par, [-1], lengths=lens)
    assert lib.sb_kernel_launch_count() == n0
    # empty calls do nothing and succeed
    e = sess.kv_cache(0, 2, 8, 32)
    sess.kv_cache_write(e, z((0,), "i32"), z((0, 1, 2, 32)), z((0, 1, 2, 32)))
    sess.kv_cache_attention(e, z((0,), "i32"), z((0, 1, 2, 32)), z((0, 1, 2, 32)))
    e = sess.kv_cache(2, 2, 0, 32, "int8")
    w(e)
    o = put(sess, np.ones((2, 1, 4, 32), np.float32))
    sess.kv_cache_attention(e, pos, q, o)
    assert not o.to_host().any()
    b(z((0, 9)), z((0, 2)), z((0, 2)), z((0, 2), "i32"), z((0, 2), "i32"))
    r([], par, [])
    r([z((0, 4))], z((0, 2), "i32"), [1])
    assert lib.sb_kernel_launch_count() == n0
    other.close()


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run(sess):
    """The same call gives the same bits, alone, between other calls and from
    two sessions at once."""
    rng = np.random.default_rng(8)
    other = S.B200Session(device=0, precision="fp32")
    got = []
    for s in (sess, other):
        cache, arrays, scales = make_cache(s, np.random.default_rng(1), (3, 4, 900, 64), "int8")
        q = put(s, rand(np.random.default_rng(2), (3, 20, 8, 64)))
        pos = put(s, np.int32([850, 3, 400]))
        lg = put(s, rand(np.random.default_rng(3), (12, 5000)))
        sc = put(s, -np.abs(rand(np.random.default_rng(4), (3, 4))))
        got.append((s, cache, q, pos, lg, sc))
    outs = []
    for _ in range(3):
        for s, cache, q, pos, lg, sc in got:
            o, osc, op, ot = s.zeros((3, 20, 8, 64)), s.zeros((3, 4)), s.zeros((3, 4), "i32"), s.zeros((3, 4), "i32")
            s.kv_cache_attention(cache, pos, q, o)
            s.beam_select(lg, sc, osc, op, ot)
            outs.append((o, osc, op, ot))
    first = [b.to_host() for b in outs[0]]
    for o in outs[1:]:
        for a, b in zip(first, o):
            assert np.array_equal(a, b.to_host())
    other.close()


@pytest.mark.gpu
def test_captured_and_replayed(sess):
    """A write, attention, selection and reorder captured on the session stream
    and replayed on new inputs equal the calls made one by one."""
    import torch
    G, W, H, T, D, V = 2, 3, 2, 50, 64, 300
    N = G * W
    rng = np.random.default_rng(3)
    dev = torch.device("cuda:0")
    t = {"k": torch.zeros(N, 2, H, D, device=dev), "v": torch.zeros(N, 2, H, D, device=dev),
         "q": torch.zeros(N, 2, 2 * H, D, device=dev), "out": torch.zeros(N, 2, 2 * H, D, device=dev),
         "pos": torch.zeros(N, dtype=torch.int32, device=dev), "lg": torch.zeros(N, V, device=dev),
         "sc": torch.zeros(G, W, device=dev), "par": torch.zeros(G, W, dtype=torch.int32, device=dev),
         "tok": torch.zeros(G, W, dtype=torch.int32, device=dev)}
    b = {k: sess.wrap_torch(x) for k, x in t.items()}
    cache = sess.kv_cache(N, H, T, D, "int8")

    def step():
        sess.kv_cache_write(cache, b["pos"], b["k"], b["v"])
        sess.kv_cache_attention(cache, b["pos"], b["q"], b["out"])
        sess.beam_select(b["lg"], b["sc"], b["sc"], b["par"], b["tok"])
        sess.beam_reorder(cache.buffers(), b["par"], [2] * 4)

    def feed(seed):
        r = np.random.default_rng(seed)
        for k in ("k", "v", "q", "lg", "sc"):
            t[k].copy_(torch.from_numpy(rand(r, tuple(t[k].shape))))
        t["pos"].copy_(torch.from_numpy(r.integers(0, T - 2, N).astype(np.int32)))
        torch.cuda.synchronize()

    def results():
        sess.synchronize()
        return [t[k].cpu().numpy() for k in ("out", "sc", "par", "tok")] + [x.to_host() for x in cache.buffers()]


    want = []
    for seed in range(3):
        feed(seed)
        step()
        want.append(results())
    cache.release()
    cache = sess.kv_cache(N, H, T, D, "int8")
    sess.synchronize()
    stream = torch.cuda.ExternalStream(sess.cuda_stream, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step()
    for seed in range(3):
        feed(seed)
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        for a, c in zip(results(), want[seed]):
            assert np.array_equal(a, c)
    del g


@pytest.mark.gpu
@pytest.mark.parametrize("kind,n_tok", [("f32", 1), ("f32", 12), ("bf16", 1), ("int8", 5), ("int8", 20)])
def test_each_attention_kernel_captured(sess, kind, n_tok):
    """The widest splits of every kernel inside a graph, with positions that change between replays."""
    import torch
    N, H, T, D = 1, 2, 5000, 64
    rng = np.random.default_rng(n_tok)
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    k, v = values(arrays, scales)
    q = rand(rng, (N, n_tok, H, D))
    pos = torch.zeros(N, dtype=torch.int32, device="cuda")
    hq, hp, out = put(sess, q), sess.wrap_torch(pos), sess.zeros(q.shape)
    sess.synchronize()
    stream = torch.cuda.ExternalStream(sess.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        sess.kv_cache_attention(cache, hp, hq, out)
    for at in (0, 4000, 31):
        pos.fill_(at)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        ref, dots, vmax, live = R.attention(k, v, [at], q, 1 / math.sqrt(D))
        assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, "f32")).all()
    del g


@pytest.mark.gpu
@pytest.mark.parametrize("src,group", [("f32", 1), ("bf16", 4), ("bf16", 16)])
def test_int8_scales_copied_by_other_lanes(sess, src, group):
    """Few rows over int8 caches of many steps: every lane reads scales that other lanes of its warp copied.  Equal
    bits from call to call, and the definition's values."""
    rng = np.random.default_rng(group)
    N, H, T, D = 6, 4, 1500, 64
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), "int8")
    for s in scales:  # a scale taken from another place would show
        s *= np.exp2(rng.integers(-3, 4, s.shape)).astype(np.float32)
    cache = S.KVCache(cache.k, cache.v, *[put(sess, s) for s in scales])
    pos = rng.integers(0, T, N)
    q = rand(rng, (N, 1, group * H, D), src)
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, 1 / math.sqrt(D))
    hq, hp = put(sess, q, src), put(sess, np.int32(pos))
    outs = [put(sess, np.zeros(q.shape, np.float32), src) for _ in range(20)]
    for out in outs:
        sess.kv_cache_attention(cache, hp, hq, out)
    got = [out.to_host() for out in outs]
    assert (np.abs(got[0] - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()
    assert all(np.array_equal(g, got[0]) for g in got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_tok,G,D", [(1, 8, 64), (9, 1, 64), (16, 1, 128), (4, 4, 48), (20, 1, 64), (33, 4, 128),
                                       (64, 3, 64), (10, 1, 256)])
def test_bf16_probabilities_keep_their_bits(sess, kind, n_tok, G, D):
    """Values that cancel: what the probabilities' rounding leaves out stands beside an output near zero.  The bound
    is elementwise: the output's own rounding (half a bf16 step of the element), the evaluation in f32 (see
    attention_bound), and what a bf16 call may leave out of each probability: 2^-16, or 2^-11 over int8 caches,
    times at most the largest value."""
    rng = np.random.default_rng(n_tok + D)
    N, H, T = 3, 2, 90
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    arrays[1] = np.where(np.arange(T)[:, None] % 2, 100, -100).astype(arrays[1].dtype) * np.ones_like(arrays[1])
    if scales:
        scales[1][:] = 0.01
    cache = S.KVCache(*([put(sess, a, kind) for a in arrays] + [put(sess, s) for s in scales]))
    q = rand(rng, (N, n_tok, G * H, D), "bf16")
    pos, scale = [6, 0, 23], 0.01 if not scales else 0.001
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, scale)
    out = put(sess, np.zeros(q.shape, np.float32), "bf16")
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, "bf16"), out, scale=scale)
    left = (2.0 ** -11 if kind == "int8" else 2.0 ** -16) * vmax[..., None]
    bound = attention_bound(dots, vmax, live, D, ref, "f32") + left
    assert (np.abs(out.to_host() - ref) <= bound * (1 + UBF) + UBF * np.abs(ref)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("V", [65, 5000])
@pytest.mark.parametrize("W", [1, 3, 8])
def test_beam_select_zeros_of_both_signs_are_equal(sess, kind, V, W):
    """-0 and +0 among the best logits, side by side (one lane has both) and far apart, in both orders: each token
    once, the lower token first."""
    rng = np.random.default_rng(V + W)
    for zeros in ([-0.0, 0.0], [0.0, -0.0], [-0.0, 0.0, -0.0, 0.0, 0.0, -0.0]):
        for step in (1, 9):
            x = -1 - rng.random((W, V)).astype(np.float32)
            x[:, 3:3 + step * len(zeros):step] = zeros
            x[0, 1] = -0.0
            x[0, V - 1] = 0.0
            x = R.bf16_round(x) if kind == "bf16" else x
            for scores in (np.zeros((1, W)), -np.arange(W)[None]):
                check_select(sess, x, np.float32(scores), np.zeros((1, W), np.int32), -1, kind)
    check_select(sess, np.where(rng.random((W, V)) < 0.5, np.float32(-0.0), np.float32(0)), np.zeros((1, W), np.float32),
                 np.zeros((1, W), np.int32), -1, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("W,V,runs", [(1, 9000, [(0, 2048)]), (2, 40000, [(0, 33000)]), (4, 70000, [(0, 69990)]),
                                      (16, 5000, [(0, 1024), (3000, 4100)]), (16, 2100, [(0, 2099)]),
                                      (3, 6001, [(5, 5990)])])
def test_beam_select_runs_of_nan(sess, kind, W, V, runs):
    """A run of NaN logits long enough that a lane's first values are NaN altogether, before, between and behind
    finite ones: each counts as -inf, the other tokens as ever."""
    x = (np.random.default_rng(V).standard_normal((2 * W, V)) * 2).astype(np.float32)
    x = R.bf16_round(x) if kind == "bf16" else x
    for a, b in runs:
        x[::2, a:b] = np.nan
    check_select(sess, x, -np.arange(2 * W, dtype=np.float32).reshape(2, W) / 8, np.zeros((2, W), np.int32), -1, kind)


def near_values(rng, G, W, V, gap):
    """Groups whose last place is between beam 0's two best, which are equal, and the second best of the last beam,
    `gap` of the value away (up to the scores' rounding, 2^-24): logits [G, W, V] and scores [G, W].  The other
    beams' best are clearly ahead of both, all else is clearly behind."""
    x = rng.standard_normal((G, W, V)).astype(np.float32)
    s = np.zeros((G, W), np.float32)
    for g in range(G):
        a, b = rng.choice(V, 2, replace=False)
        x[g, 0, [a, b]] = 8.5
        for w in range(1, W):
            t = rng.choice(V, 2, replace=False)
            x[g, w, t] = 12.0, 8.25
        lse = np.log(np.exp(x[g].astype(np.float64)).sum(1))
        s[g, W - 1] = 8.5 - lse[0] + gap[g] - (8.25 - lse[W - 1])
        s[g, 1:W - 1] = 0.5 - np.arange(W - 2) / 16
    return x, s


@pytest.mark.gpu
@pytest.mark.parametrize("W,V", [(2, 3000), (2, 50304), (4, 4097), (8, 1500)])
def test_beam_select_order_at_the_last_place(sess, W, V):
    """Two equal candidates of one beam at the cut, and another beam's behind them that f64 sums put before or after
    them by less than f32 sums can tell."""
    rng = np.random.default_rng(W + V)
    G = 48 if V < 9000 else 12
    x, s = near_values(rng, G, W, V, rng.uniform(-6e-7, 6e-7, G))
    ref = R.beam_select(x.reshape(G * W, V), s)
    assert len(set(ref[1][:, -1])) == 2  # either beam has the last place somewhere
    check_select(sess, x.reshape(G * W, V), s, np.zeros((G, W), np.int32), -1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rise", [("f32", 30.0), ("bf16", 8.0), ("f32", 2.0)])
def test_beam_select_scores_of_rising_logits(sess, kind, rise):
    """4M logits that rise along the vocabulary: a lane's maximum moves with each of its pieces, and the scores stay
    within the 4e-6 that is said of them (before their own rounding), the order that of 64-bit sums."""
    W, V = 16, 1 << 22
    rng = np.random.default_rng(5)
    x = (np.linspace(0, rise, V) + rng.random((W, 1))).astype(np.float32)
    if kind == "bf16":
        x = R.bf16_round(x)
    s = -np.sort(rng.random((1, W))).astype(np.float32) / 64
    ref = R.beam_select(x, s)
    osc, par, tok = sess.zeros((1, W)), sess.zeros((1, W), "i32"), sess.zeros((1, W), "i32")
    sess.beam_select(put(sess, x, kind), put(sess, s), osc, par, tok)
    assert np.array_equal(par.to_host(), ref[1])
    assert np.array_equal(tok.to_host(), ref[2])
    assert (np.abs(osc.to_host() - ref[0]) <= U32 * np.abs(ref[0]) + 4e-6).all()


@pytest.mark.gpu
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", [(1, 1, 32), (1, 1, 64), (1, 4, 128), (6, 2, 64), (12, 1, 48), (20, 2, 64),
                                       (33, 4, 128), (2, 1, 256)])
@pytest.mark.parametrize("e", [-112, 100])
def test_attention_of_extreme_values(sess, src, n_tok, G, D, e):
    """Value scales near the ends of f32's range: outputs of that size, by every kernel."""
    rng = np.random.default_rng(n_tok + D)
    N, H, T = 2, 2, 170
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), "int8")
    scales[1] = np.ldexp(scales[1], e)
    cache.v_scale = put(sess, scales[1])
    q = rand(rng, (N, n_tok, G * H, D), src)
    pos = [T - n_tok, 17]
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, 1 / math.sqrt(D))
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, src)).all()


FAR_SHAPES = [(1, 1, 64), (1, 1, 32), (1, 4, 128), (6, 1, 64), (7, 2, 48), (12, 1, 64), (4, 3, 128), (20, 2, 64),
              (33, 4, 128), (64, 3, 64), (2, 1, 256)]


def weighted_bound(k, v, pos, q, scale, parents, src, kind):
    """The 64-bit result, and how far an evaluation may be from it where value rows differ by orders of magnitude: a
    relative error of e in each probability (see attention_bound) moves an element by at most 2 e sum p |v|, the sum
    over the keys that the token sees; what a bf16 call may leave out of a probability, and its output's rounding.
    f16 products keep 2^-30 of the row's largest p |v|, which is within e of the row's largest sum."""
    ref, dots, _, live = R.attention(k, v, pos, q, scale, parents)
    total = R.attention(k, np.abs(v), pos, q, scale, parents)[0].max(-1)
    e = 2 * (q.shape[-1] + 4) * U32 * dots + (live + 64) * U32
    b = 2 * e * total
    if src == "bf16":
        b = b + (2.0 ** -11 if kind == "int8" else 2.0 ** -16) * total
    b = b[..., None] * np.ones_like(ref)
    return ref, b * (1 + UBF) + UBF * np.abs(ref) if src == "bf16" else b


@pytest.mark.gpu
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", [c for c in FAR_SHAPES if c[0] > 1])
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e30, 1e38, 1e-30])
def test_attention_value_scales_of_unseen_tokens(sess, src, n_tok, G, D, ratio):
    """Drafted tokens whose int8 value rows are larger or smaller than all others by orders of magnitude (1e38: as an
    infinity is stored), early and late in a tree: the tokens that do not attend to them give what they gave."""
    rng = np.random.default_rng(n_tok + D)
    N, H, T, pos = 3, 2, 230, [150, 0, 61]
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), "int8")
    far = {n_tok // 2, n_tok - 1}
    for n in range(N):
        for t in far:
            scales[1][n, :, pos[n] + t] *= np.float32(ratio)
            arrays[1][n, :, pos[n] + t] //= 2
    cache.v_scale, cache.v = put(sess, scales[1]), put(sess, arrays[1])
    q = rand(rng, (N, n_tok, G * H, D), src)
    parents = np.full((N, n_tok), -1, np.int32)
    parents[:, n_tok // 2 + 1:n_tok - 1] = 0
    k, v = values(arrays, scales)
    ref, bound = weighted_bound(k, v, pos, q, 1 / math.sqrt(D), parents, src, "int8")
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out, parents=put(sess, parents))
    assert (np.abs(out.to_host() - ref) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", FAR_SHAPES)
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9, 1e20])
@pytest.mark.parametrize("at", [0, 100, 399])
def test_attention_value_scales_of_little_weight(sess, src, n_tok, G, D, ratio, at):
    """One int8 value row larger than the others by orders of magnitude at a probability that undoes it, before,
    between and behind the others: all of them count."""
    rng = np.random.default_rng(n_tok + D + at)
    N, H, T, pos = 2, 2, 480, [400, 400]
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), "int8")
    scales[0] *= 0.1
    scale = 1 / math.sqrt(D)
    q = np.repeat(np.repeat(rand(rng, (N, 1, H, D)), n_tok, 1), G, 2)
    q = R.bf16_round(q + 0.01 * rand(rng, q.shape))
    u = q[:, 0, ::G]
    arrays[0][:, :, at] = -np.rint(u * 127 / np.abs(u).max(-1, keepdims=True))
    scales[0][:, :, at] = -np.log(ratio) / (scale * (u * arrays[0][:, :, at]).sum(-1))
    scales[1][:, :, at] *= np.float32(ratio)
    cache = S.KVCache(*([put(sess, a) for a in arrays] + [put(sess, s) for s in scales]))
    k, v = values(arrays, scales)
    ref, bound = weighted_bound(k, v, pos, q, scale, None, src, "int8")
    out = put(sess, np.zeros(q.shape, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    assert (np.abs(out.to_host() - ref) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", [(1, 1, 32), (2, 2, 64), (12, 1, 64), (20, 2, 64), (33, 4, 128), (2, 1, 256)])
def test_attention_of_scores_that_are_nan_or_all_lowest(sess, kind, src, n_tok, G, D):
    """A query with a NaN gives NaN, and so do scores of -inf throughout (their softmax is 0 / 0); the other rows
    their values; a row without keys stays zero."""
    rng = np.random.default_rng(n_tok + D)
    N, H, T, pos = 3, 2, 120, [90, 0, -1]
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    q = rand(rng, (N, n_tok, G * H, D), src)
    k, v = values(arrays, scales)
    ref, dots, vmax, live = R.attention(k, v, pos, q, 1 / math.sqrt(D))
    bad = np.zeros(q.shape[:3], bool)
    bad[:, n_tok // 2, 0] = True
    q[:, n_tok // 2, 0, 5] = np.nan
    if not scales:
        arrays[0][0, 1] = -np.inf
        q[0, :, G:] = np.abs(q[0, :, G:]) + 1
        bad[0, :, G:] = True
        cache.k = put(sess, arrays[0], kind)
    out = put(sess, np.full(q.shape, 7.0, np.float32), src)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    got = out.to_host()
    assert np.isnan(got[bad & (live > 0)]).all()
    assert not got[live == 0].any()
    ok = ~bad
    assert (np.abs(got - ref) <= attention_bound(dots, vmax, live, D, ref, src))[ok].all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok,G,D", [(1, 1, 32), (1, 2, 64), (7, 1, 64), (12, 1, 64), (20, 2, 64), (33, 4, 128),
                                       (2, 1, 256)])
def test_attention_of_nan_at_no_weight(sess, kind, src, n_tok, G, D):
    """A NaN value row that a token attends to reaches it whatever its probability, one that rounds to 0 too, in
    full steps of keys as in the last."""
    rng = np.random.default_rng(n_tok + D)
    N, H, T, pos = 2, 1, 400, [370, 20]
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    q = np.abs(rand(rng, (N, n_tok, G * H, D), src)) + 1
    q = R.bf16_round(q)
    for n in range(N):  # scores of some -1000 for the first key and the last before the drafted ones
        at = [0, pos[n] - 1][n]
        arrays[0][n, :, at] = -100
        if scales:
            scales[0][n, :, at] = 1
            scales[1][n, :, at] = np.nan
        else:
            arrays[1][n, :, at] = np.nan
    got = _attend(sess, arrays, scales, kind, pos, q, src, np.full((N, n_tok), -1, np.int32))
    assert np.isnan(got).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_tok,D", [(1, 64), (20, 64), (1, 256)])
def test_attention_at_the_largest_scales(sess, lib, kind, n_tok, D):
    """A scale whose product with log2(e) passes f32's range is refused; the largest that fits gives queries of zero
    the mean of the values."""
    rng = np.random.default_rng(D)
    cache, arrays, scales = make_cache(sess, rng, (1, 2, 50, D), kind)
    k, v = values(arrays, scales)
    q = np.zeros((1, n_tok, 2, D), np.float32)
    out, pos = sess.zeros(q.shape), put(sess, np.int32([20]))
    n0 = lib.sb_kernel_launch_count()
    for scale in (2.4e38, 3.4e38, -2.4e38, float("inf")):
        with pytest.raises(S.B200Error) as e:
            sess.kv_cache_attention(cache, pos, put(sess, q), out, scale=scale)
        assert e.value.code == 3
    assert lib.sb_kernel_launch_count() == n0
    ref, dots, vmax, live = R.attention(k, v, [20], q, 1.0)
    for scale in (2.3e38, -2.3e38):
        sess.kv_cache_attention(cache, pos, put(sess, q), out, scale=scale)
        assert (np.abs(out.to_host() - ref) <= attention_bound(dots, vmax, live, D, ref, "f32")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("src", ["f32"])
def test_attention_sums_over_long_caches(sess, kind, src):
    """f32 rows on the tensor cores over many long caches, which are split no further to fill the SMs: the sums, which
    truncate, stay short.  32 tiles of 64 keys take 12 additions each, which fall short by half a step of f32 on the
    average, 2^-24 of the sum at most: 384 of them 2.3e-5 of the outputs."""
    rng = np.random.default_rng(3)
    N, H, T, D, n_tok = 10, 8, 24000, 64, 9
    cache, arrays, scales = make_cache(sess, rng, (N, H, T, D), kind)
    q = rand(rng, (N, n_tok, H, D), src)
    pos = [T - n_tok] * N
    out = sess.zeros(q.shape)
    sess.kv_cache_attention(cache, put(sess, np.int32(pos)), put(sess, q, src), out)
    some = slice(0, None, 4)
    k, v = values([a[some] for a in arrays], [s[some] for s in scales])
    ref = R.attention(k, v, pos[some], q[some], 1 / math.sqrt(D))[0]
    got = out.to_host()[some].astype(np.float64)
    assert np.linalg.norm(got - ref) <= 384 * U32 * np.linalg.norm(ref)
