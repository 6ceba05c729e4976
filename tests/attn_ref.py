"""Plain 64-bit forms of the operators of ops.dot_attention / embedding / newton_schulz, with the error bounds their tests use.

Every bound counts roundings: u32 = 2^-24 per fp32 operation or sum step, u16 = 2^-8 per value rounded to bf16 (0 for fp32)."""
import numpy as np

U32 = 2.0 ** -24
U16 = 2.0 ** -8
TINY = 2.0 ** -126                                                      # smallest normal fp32 and bf16 number
ATTENDED = -1e8


def attention(q, k, v, bias=None, key_sizes=None, query_sizes=None, scale=None, dout=None, bf16=False):
    """float64 arrays q [B,Nq,H,D], k, v [B,Nk,G,D] -> dict of (value, bound) for out and, with dout, dq, dk, dv.

    Scores: an fp32 dot product of D terms is off by (D + 2) u32 sum |q k|; scaling, bias, the change to base 2 and the subtraction of the
    row's lse are a few more roundings of numbers no larger than |z| + |lse|.  A numerator's relative error is the absolute error of
    its exponent, the row's normalisation has at most the largest of them: rho = 2 max_j e_ij.  Sums over n terms: n u32 of the sum
    of magnitudes.  bf16: results are rounded; P and dz enter the second products as two numbers each, rounded to
    one for many rows (beyond 1024 nodes) without a mask; the saved `out` (inside delta) is two numbers.
    Underflow: an exponential below 2^-126 may be flushed to zero (its weight at most TINY off), and so may the two low parts of a dz
    that is computed as three bf16 (2 TINY)."""
    B, Nq, H, D = q.shape
    Nk, G = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    ur = U16 if bf16 else 0.0
    up = 0.0 if not bf16 else U16 if bias is None and min(Nq * (H // G), Nk) > 64 and max(Nq, Nk) > 1024 else U16 ** 2
    z0 = lambda x: np.zeros(x.shape)
    res = {"out": [z0(q), z0(q)]}
    if dout is not None:
        res.update(dq=[z0(q), z0(q)], dk=[z0(k), z0(k)], dv=[z0(k), z0(k)])
    for b in range(B):
        nk = Nk if key_sizes is None else int(np.clip(key_sizes[b], 0, Nk))
        nq = Nq if query_sizes is None else int(np.clip(query_sizes[b], 0, Nq))
        for h in range(H):
            g = h // (H // G)
            Q, K, V = q[b, :nq, h], k[b, :nk, g], v[b, :nk, g]
            bm = np.zeros((nq, nk)) if bias is None else bias[b if bias.shape[0] > 1 else 0, :nq, :nk]
            seen = bm > ATTENDED
            s = scale * (Q @ K.T)
            z = np.where(seen, s + bm, -np.inf)
            top = np.where(seen.any(1), z.max(1, initial=-np.inf), 0.0)[:, None]
            p = np.exp(z - top)
            l = p.sum(1, keepdims=True)
            p = p / np.where(l > 0, l, 1.0)
            lse = np.where(l > 0, np.log(np.where(l > 0, l, 1.0)) + top, 0.0)
            zf = np.where(seen, z, 0.0)
            e = U32 * ((D + 4) * abs(scale) * (abs(Q) @ abs(K).T) + 6 * abs(zf) + 6 * abs(lse) + 8)
            rho = 2 * np.where(seen, e, 0.0).max(1, initial=0.0)[:, None] + (nk + 16) * U32
            out = p @ V
            pv = p @ abs(V)
            e_sum = (rho + up) * pv + (nk + 8) * U32 * pv + TINY * abs(V).sum(0)
            e_out = e_sum + ur * (abs(out) + e_sum)
            res["out"][0][b, :nq, h] = out
            res["out"][1][b, :nq, h] = e_out
            if dout is None:
                continue
            dO = dout[b, :nq, h]
            dp, delta = dO @ V.T, (dO * out).sum(1, keepdims=True)
            ds = p * (dp - delta)
            dpa = abs(dO) @ abs(V).T
            e_delta = (D + 4) * U32 * (abs(dO) * abs(out)).sum(1, keepdims=True) + (abs(dO) * (e_sum + ur ** 2 * (abs(out) + e_sum))).sum(1, keepdims=True)
            e_ds = p * (rho * (abs(dp) + abs(delta)) + (D + 4) * U32 * dpa + e_delta + 4 * U32 * (abs(dp) + abs(delta)))
            e_ds = e_ds + TINY * (abs(dp) + abs(delta) + 2)
            e_use = e_ds + up * (abs(ds) + e_ds)
            dq, dk, dv = scale * (ds @ K), scale * (ds.T @ Q), p.T @ dO
            adds = abs(ds) + e_ds
            res["dq"][0][b, :nq, h] = dq
            res["dq"][1][b, :nq, h] = abs(scale) * (e_use @ abs(K) + (nk + 8) * U32 * (adds @ abs(K)))
            n = nq * (H // G)
            res["dk"][0][b, :nk, g] += dk
            res["dk"][1][b, :nk, g] += abs(scale) * (e_use.T @ abs(Q) + (n + 8) * U32 * (adds.T @ abs(Q)))
            res["dv"][0][b, :nk, g] += dv
            res["dv"][1][b, :nk, g] += (p * (rho + up) + 3 * TINY).T @ abs(dO) + (n + 8) * U32 * (p.T @ abs(dO))
    for name in ("dq", "dk", "dv"):
        if name in res:
            res[name][1] += ur * (abs(res[name][0]) + res[name][1])
    return {n: tuple(x) for n, x in res.items()}


def embedding_grad(ids, dout, rows, scale, bf16=False):
    """(value, bound) of scale * sum of dout over the tokens of each row: n additions, one product, one rounding."""
    ids = ids.reshape(-1)
    d = dout.reshape(len(ids), dout.shape[-1])
    ok = (ids >= 0) & (ids < rows)
    value, mags, count = np.zeros((rows, d.shape[1])), np.zeros((rows, d.shape[1])), np.zeros((rows, 1))
    np.add.at(value, ids[ok], d[ok])
    np.add.at(mags, ids[ok], abs(d[ok]))
    np.add.at(count, ids[ok], 1.0)
    value *= scale
    return value, (count + 2) * U32 * mags * abs(scale) + (U16 if bf16 else 0.0) * abs(value) * 1.001


def newton_schulz(x, steps=5, eps=1e-7, coefficients=(3.4445, -4.7750, 2.0315)):
    a, b, c = coefficients
    x = x / (np.sqrt((x * x).sum()) + eps)
    if x.shape[0] > x.shape[1]:
        return newton_schulz_steps(x.T, steps, a, b, c).T
    return newton_schulz_steps(x, steps, a, b, c)


def newton_schulz_steps(x, steps, a, b, c):
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def within(got, value, bound, what):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == value.shape, "%s: shape %s, expected %s" % (what, got.shape, value.shape)
    err = np.abs(got - value)
    bad = ~(err <= bound + 1e-38)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, err / (bound + 1e-38), 0.0)), err.shape)
        raise AssertionError("%s: %d of %d outside the bound; worst at %s: got %.9g, expected %.9g, off %.3g, bound %.3g"
                             % (what, bad.sum(), bad.size, i, got[i], value[i], err[i], bound[i]))
