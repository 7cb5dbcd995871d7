"""Plain numpy restatement, in 64 bits, of the decoding operators
(include/sheaf_b200.h, "decoding operators").  Tests only."""
import numpy as np


def bf16_round(x):
    """f32 values rounded to nearest-even bf16, as f32 (finite values and infinities)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32).reshape(np.shape(x))


def quantise(x):
    """(codes int8, scale f32) of rows [..., D]: scale = max|x| / 127 in f32,
    code = x / scale to the nearest integer, ties to even (the f64 quotient of
    two f32 values is within 2^-53 of the exact one, which cannot cross a tie:
    an exact quotient that is not a tie differs from it by at least 2^-25)."""
    big = np.finfo(np.float32).max
    x = np.clip(np.nan_to_num(np.asarray(x, np.float32), nan=0.0, posinf=big, neginf=-big), -big, big)
    scale = (np.abs(x).max(-1).astype(np.float64) / 127.0).astype(np.float32)
    s = scale.astype(np.float64)[..., None]
    q = np.rint(np.divide(x.astype(np.float64), s, out=np.zeros(x.shape), where=s > 0))
    return np.clip(q, -127, 127).astype(np.int8), scale


def write(cache, scale, positions, x):
    """In place; cache [N, H, T, D] (f32 values, bf16 values as f32 when `scale`
    is "bf16", or int8 codes), x [N, S, H, D]."""
    N, S = x.shape[:2]
    T = cache.shape[2]
    for n in range(N):
        for s in range(S):
            t = int(positions[n]) + s
            if positions[n] < 0 or t >= T:
                continue
            if isinstance(scale, np.ndarray):
                cache[n, :, t], scale[n, :, t] = quantise(x[n, s])
            else:
                cache[n, :, t] = bf16_round(x[n, s]) if scale == "bf16" else x[n, s]


def ancestors(parents, S):
    """[S, S] bool: token s attends to token j (itself and its ancestors)."""
    seen = np.zeros((S, S), bool)
    for s in range(S):
        j = s
        while True:
            seen[s, j] = True
            p = j - 1 if parents is None else int(parents[j])
            if not 0 <= p < j:
                break
            j = p
    return seen


def attention(k, v, positions, q, scale, parents=None):
    """k, v [N, H, T, D] values (f64), q [N, S, Hq, D]; returns (out, bound)
    where bound[n, s, h] = max over the seen keys of sum_d |q_d k_d| * scale and
    of |v|, for error bounds."""
    N, S, Hq, D = q.shape
    H, T = k.shape[1:3]
    out = np.zeros(q.shape)
    dots, vmax, live = np.zeros((N, S, Hq)), np.zeros((N, S, Hq)), np.zeros((N, S, Hq), int)
    for n in range(N):
        pos = int(positions[n])
        if pos < 0:
            continue
        seen = ancestors(None if parents is None else parents[n], S)
        for s in range(S):
            at = [t for t in range(min(pos, T))] + [pos + j for j in range(S) if seen[s, j] and pos + j < T]
            if not at:
                continue
            for h in range(Hq):
                kk, vv = k[n, h // (Hq // H), at], v[n, h // (Hq // H), at]
                z = scale * (kk @ q[n, s, h].astype(np.float64))
                e = np.exp(z - z.max())
                out[n, s, h] = (e / e.sum()) @ vv
                dots[n, s, h] = (np.abs(kk) @ np.abs(q[n, s, h].astype(np.float64))).max() * abs(scale)
                vmax[n, s, h] = np.abs(vv).max()
                live[n, s, h] = len(at)
    return out, dots, vmax, live


def beam_select(logits, scores, finished=None, eos=-1):
    """logits [G * W, V], scores [G, W] -> scores (f64), parents, tokens, finished."""
    G, W = scores.shape
    V = logits.shape[1]
    z = np.asarray(logits, np.float64).reshape(G, W, V).copy()
    z[np.isnan(z)] = -np.inf
    outs = []
    for g in range(G):
        cands = []
        for w in range(W):
            top = z[g, w].max()
            with np.errstate(all="ignore"):
                lse = top + np.log(np.exp(z[g, w] - top).sum())
            if not np.isfinite(scores[g, w]) or not np.isfinite(lse) and not (eos >= 0 and finished[g, w]):
                row = [(-np.inf, w, v) for v in range(min(W, V))]
            elif eos >= 0 and finished[g, w]:
                row = [(float(scores[g, w]), w, eos)] + [(-np.inf, w, v) for v in range(V) if v != eos][:W - 1]
            else:
                order = np.argsort(-z[g, w], kind="stable")[:W]
                row = [(float(scores[g, w]) + (z[g, w, v] - lse), w, int(v)) for v in order]
            cands += row
        best = sorted(range(len(cands)), key=lambda i: (-cands[i][0], i))[:W]
        outs.append([cands[i] + (int(eos >= 0 and bool(finished[g, cands[i][1]] or cands[i][2] == eos)),)
                     for i in best])
    a = np.array(outs, np.float64).reshape(G, W, 4)
    return a[..., 0], a[..., 1].astype(np.int32), a[..., 2].astype(np.int32), a[..., 3].astype(np.int32)


def reorder(state, parents, axis, lengths=None):
    """A new array: `state` after beam_reorder."""
    G, W = parents.shape
    out = state.copy()
    for g in range(G):
        for j in range(W):
            p = int(parents[g, j])
            if not 0 <= p < W:
                continue
            i = ()
            if axis >= 0 and lengths is not None:
                n = max(0, min(int(lengths[g * W + p]), state.shape[axis]))
                i = (slice(None),) * (axis - 1) + (slice(0, n),)
            out[(g * W + j,) + i] = state[(g * W + p,) + i]
    return out
