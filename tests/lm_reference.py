"""The definitions of token_logprob, rotary, qk_norm_rotary and the Newton-Schulz orthogonalisation in 64 bits
(numpy), with the bounds on a kernel's rounding that the tests use."""
import numpy as np

U = 2.0 ** -24          # half an ulp of fp32, relative


# ---- token_logprob ----------------------------------------------------------------------------------
def token_logprob(x, token, temperature=1.0, top=0):
    """x [rows, C] float32, token [rows]. Returns a dict of float64 arrays (top_index int)."""
    z = x.astype(np.float64) / float(np.float32(temperature))
    rows, C = z.shape
    out = {k: np.zeros(rows) for k in ("logprob", "entropy", "log_norm", "shift")}
    out["p"], out["logp"] = np.zeros_like(z), np.full_like(z, -np.inf)
    out["top_logprob"], out["top_index"] = np.zeros((rows, top)), np.zeros((rows, top), dtype=np.int64)
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = z[r].max()
            if np.isnan(z[r]).any() or m == np.inf:
                for k in ("logprob", "entropy", "log_norm"):
                    out[k][r] = np.nan
                out["p"][r] = out["logp"][r] = np.nan
                if not 0 <= token[r] < C:
                    out["logprob"][r] = 0.0
            elif m == -np.inf:
                out["logprob"][r] = out["log_norm"][r] = -np.inf
                if not 0 <= token[r] < C:
                    out["logprob"][r] = 0.0
            else:
                log_s = np.log(np.exp(z[r] - m).sum())
                L, lp = m + log_s, (z[r] - m) - log_s     # not z - L: far from 0 L has no digits left for it
                p = np.exp(lp)
                out["shift"][r], out["log_norm"][r], out["p"][r], out["logp"][r] = m, L, p, lp
                out["entropy"][r] = -np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0).sum()
                out["logprob"][r] = lp[token[r]] if 0 <= token[r] < C else 0.0
            if top:
                keyed = np.where(np.isnan(x[r]), -np.inf, x[r].astype(np.float64))
                order = np.lexsort((np.arange(C), np.isnan(x[r]), -keyed))[:top]
                live = ~np.isnan(x[r][order])
                out["top_index"][r] = np.where(live, order, -1)
                out["top_logprob"][r] = np.where(live, out["logp"][r][order], np.nan)
    return out


def token_logprob_grad(ref, token, temperature, gl, gh, gn):
    """d/dx in 64 bits from token_logprob()'s result; NULL upstream gradients are zeros."""
    p, logp, H = ref["p"], ref["logp"], ref["entropy"][:, None]
    rows, C = p.shape
    valid = (token >= 0) & (token < C)
    gl = np.where(valid, gl, 0.0)
    with np.errstate(all="ignore"):
        slope = np.where(p > 0, np.where(p > 0, logp, 0.0) + H, 0.0)
        g = p * (gn[:, None] - gl[:, None] - gh[:, None] * slope)
    for r in np.nonzero(valid & (ref["log_norm"] != -np.inf))[0]:
        g[r, token[r]] += gl[r]
    return g / float(np.float32(temperature))


def log_sum_bound(ref, C):
    """Relative error of S = sum exp(z - m), i.e. absolute error of log S: an exponential's 2^-22; three
    roundings of its argument t, whose mean over the distribution is at most log2(C) and a little (t * U * 3 * ln 2);
    at most 64 additions one after the other in a thread for the sizes tested, then 5 + 4 + 3 merges, each with
    one more exponential."""
    return 2.0 ** -22 * 13 + 3 * np.log(2.0) * (np.log2(C) + 2) * U + (64 + 12) * U


# ---- rotary ---------------------------------------------------------------------------------------------
def rotate(x, position, freq, interleaved=False, amplitude=1.0, sign=1.0):
    """x [..., D] float64; position broadcasts against x.shape[:-1]; freq [n] float32."""
    n = len(freq)
    a = np.broadcast_to(np.asarray(position, dtype=np.float64)[..., None] * freq.astype(np.float64),
                        x.shape[:-1] + (n,))
    c, s = np.cos(a), sign * np.sin(a)
    y = np.array(x, dtype=np.float64)
    ia, ib = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    u, v = x[..., ia], x[..., ib]
    y[..., ia] = amplitude * (u * c - v * s)
    y[..., ib] = amplitude * (u * s + v * c)
    return y


def qk_norm(x, w, epsilon):
    r = 1.0 / np.sqrt((x * x).mean(axis=-1, keepdims=True) + float(np.float32(epsilon)))
    return x * r, r, x * r * w


def qk_norm_rotary_grad(x, w, epsilon, du):
    """(dx, dw) from du = R^T dy."""
    n, r, _ = qk_norm(x, w, epsilon)
    dn = du * w
    dw = (du * n).reshape(-1, x.shape[-1]).sum(axis=0)
    return r * (dn - n * (dn * n).mean(axis=-1, keepdims=True)), dw


# ---- Newton-Schulz ----------------------------------------------------------------------------------------
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalise(u, steps=5, epsilon=1e-7):
    a, b, c = (float(np.float32(v)) for v in COEFFICIENTS)
    u = np.asarray(u, dtype=np.float64)
    x = u.T if u.shape[0] > u.shape[1] else u
    x = x / (np.linalg.norm(x) + float(np.float32(epsilon)))
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.T if u.shape[0] > u.shape[1] else x
