"""The beam decoding operators from their definitions, row by row in 64 bits (numpy)."""
import numpy as np


def seen(length, prefix, window, sinks):
    """Prefix rows and own rows that a lane with `length` cached own rows sees (own row `length`
    is the new one)."""
    at = prefix + length
    rows = [j for j in range(at + 1) if window == 0 or j < sinks or j > at - window]
    return [j for j in rows if j < prefix], [j - prefix for j in rows if j >= prefix]


def place(row, keep, capacity):
    """The cache row that own row `row` lies in."""
    return row if row < keep else keep + (row - keep) % (capacity - keep)


def lane(q, k_new, v_new, k, v, length, prefix_k, prefix_v, heads, scale, window, sinks):
    """One lane: k, v [capacity, width] receive the new row; returns the output row and the
    size of what rounding may do to it (see `bound`)."""
    width, capacity, prefix = q.size, k.shape[0], prefix_k.shape[0]
    hw = width // heads
    keep = max(0, sinks - prefix) if window else 0
    at = place(length, keep, capacity)
    k[at], v[at] = k_new.astype(np.float32).astype(k.dtype), v_new.astype(np.float32).astype(v.dtype)
    pre, own = seen(length, prefix, window, sinks)
    own = [place(r, keep, capacity) for r in own]
    kk = np.concatenate([prefix_k[pre], k[own]]).astype(np.float64).reshape(-1, heads, hw)
    vv = np.concatenate([prefix_v[pre], v[own]]).astype(np.float64).reshape(-1, heads, hw)
    qq = q.astype(np.float64).reshape(heads, hw)
    with np.errstate(invalid="ignore", over="ignore"):
        x = scale * np.einsum("hd,rhd->hr", qq, kk)
        e = np.exp(x - x.max(1, keepdims=True))
        w = e / e.sum(1, keepdims=True)
        out = np.einsum("hr,rhd->hd", w, vv).reshape(-1)
        reach = abs(scale) * np.einsum("hd,rhd->hr", abs(qq), abs(kk)).max(1)
        spread = np.repeat(bound(reach, hw, kk.shape[0])[:, None] * abs(vv).max((0, 2))[:, None], hw, 1).reshape(-1)
    return out, spread


def bound(reach, hw, rows):
    """How far a 32-bit result may be from the definition, relative to the largest |v|.  `reach`
    is the largest scale * sum |q_d k_d| of a row.  With u = 2^-24:
    * a score is a sum of hw products of a query scaled by a rounded constant: hw + 4 roundings of
      at most u * reach, and as much again from operands kept as two 11-bit halves (2^-22 each);
    * a weight is 2^(score - max) by an approximation off by at most 2^-22, and both the score and
      the maximum it is compared with carry that error: relative error 2 * dx + 2^-22, kept as two
      11-bit halves 2^-22 more;
    * weights enter the numerator and the denominator, whose sums over `rows` rows are off by at
      most rows * u each (their terms are positive, the numerator's are bounded by |v|)."""
    u = 2.0 ** -24
    dx = reach * ((hw + 4) * u + 2 * 2.0 ** -22)
    return 2 * (2 * dx + 2 * 2.0 ** -22 + rows * u) + 4 * u


def drift(q, kk, vv, heads, scale, got):
    """How far a lane's result `got` is from the definition over rows kk, vv [rows, width], as a
    sum of squares, and the sum of squares it may reach.  `bound` adds roundings up as if they were all
    alike; over many outputs they are not, and what is left is far smaller.  With u = 2^-24:
    * a weight is off by a part d_j of itself, so an output by sum_j d_j w_j (v_j - out): the d_j of
      the rows go either way, so its square is d^2 sum_j w_j^2 (v_j - out)^2, at most with |v_j| + |out|;
    * d holds the score's error.  A score is a sum of products of planes, the small ones first, whose
      sum is below 2^-8 of it; then come up to 8 sums of 16 products (head widths up to 128), each cut
      to 24 bits of what is summed so far, which is of the size x = log2(e) scale sqrt(sum (q k)^2):
      sqrt(8) 2 u x / sqrt(3) = 3.3 u x, and as much for what is cut inside a sum of 16: 7 u x;
    * and the weight's own, 8 u: its approximation 4, its planes 2, its place in the sums 2;
    * an output is a sum, a quotient and its stored value: 4 u of itself."""
    u = 2.0 ** -24
    rows, width = kk.shape
    qq = q.astype(np.float64).reshape(heads, -1)
    kk, vv = (t.astype(np.float64).reshape(rows, heads, -1) for t in (kk, vv))
    x = scale * np.einsum("hd,rhd->hr", qq, kk)
    w = np.exp(x - x.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    out = np.einsum("hr,rhd->hd", w, vv)
    size = np.log2(np.e) * abs(scale) * np.sqrt(np.einsum("hd,rhd->hr", qq ** 2, kk ** 2).max(1))
    walk = np.einsum("hr,rhd->hd", w ** 2, (abs(vv) + abs(out)) ** 2)
    may = ((7 * size + 8) * u)[:, None] ** 2 * walk + (4 * u * out) ** 2
    return ((got.reshape(heads, -1) - out) ** 2).sum(), may.sum()


def select(logits, score, done, codebook, eos, allow):
    """logits [requests, beams, vocab] -> score, token, parent, done [requests, beams]."""
    requests, beams, vocab = logits.shape
    out = (np.full((requests, beams), -np.inf), np.zeros((requests, beams), np.int64),
           np.tile(np.arange(beams), (requests, 1)), np.zeros((requests, beams), np.int64))
    for i in range(requests):
        found = []
        tokens = list(range(codebook)) + ([eos] if codebook <= eos < vocab and allow[i] else [])
        for b in range(beams):
            if done[i, b]:
                if score[i, b] > -np.inf:
                    found.append((-float(score[i, b]), b, 0.0, eos))
                continue
            x = logits[i, b, tokens].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            if not len(tokens) or x.max() == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                lse = x.max() + np.log(np.exp(x - x.max()).sum())
                c = float(score[i, b]) + (x - lse)
            found += [(-c[j], b, -x[j], t) for j, t in enumerate(tokens) if c[j] > -np.inf]
        for place_, (c, b, _, t) in enumerate(sorted(found)[:beams]):
            out[0][i, place_], out[1][i, place_], out[2][i, place_], out[3][i, place_] = -c, t, b, t == eos
    return out


def reorder(k, parent, length):
    """k [requests, beams, layers, capacity, width] -> the beams' new rows, and their lengths."""
    out, new = k.copy(), length.copy()
    requests, beams = parent.shape
    for i in range(requests):
        for b in range(beams):
            p = parent[i, b]
            if not 0 <= p < beams:
                continue
            new[i, b] = length[i, p]
            out[i, b, :, :length[i, p]] = k[i, p, :, :length[i, p]]
    return out, new
