"""Plain 64-bit forms of the norms, 8-bit codes, products and log probabilities, and the error
bounds that their tests use. numpy only; bf16 arrays travel as uint16."""
import numpy as np

from attn_reference import HALF_STEP, U, from_type, to_type

# half the distance of a type's smallest numbers, below which a rounding is no longer relative
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def norm(x, w, eps, residual=None, residual_type=None, kept=False, offset=0.0):
    """(h, y) in float64 of float64 rows: the addition in float, rounded to the residual's type
    where it is kept; y from what was kept."""
    h = x.astype(np.float32)
    if residual is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            h = h + residual.astype(np.float32)
    if kept:
        h = from_type(to_type(h, residual_type), residual_type)
    h = h.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        y = h * (1.0 / np.sqrt((h * h).sum(-1, keepdims=True) / h.shape[-1] + eps)) * (w + offset)
    return h, y


def norm_bound(y, t):
    """Of y rounded to float and then to t."""
    return np.abs(y) * (U + HALF_STEP[t]) * 1.01 + TINY[t] + 2.0 ** -150


def rows_i8(y):
    """Codes and scales of float32 rows, whole-number arithmetic deciding at the halves."""
    y = y.astype(np.float32)
    codes, scales = np.zeros(y.shape, np.int8), np.zeros(y.shape[0], np.float32)
    for r, row in enumerate(y):
        if not np.all(np.isfinite(row)):
            scales[r] = np.nan
            continue
        s = np.float32(np.float64(np.abs(row).max()) / 127)
        scales[r] = s
        if s == 0:
            continue
        n = np.rint(row.astype(np.float64) / np.float64(s))
        rest = 2 * (row.astype(np.float64) - n * np.float64(s))  # exact: 32 bits at most
        odd = n % 2 != 0
        n += (rest > s) | ((rest == s) & odd)
        n -= (rest < -s) | ((rest == -s) & odd)
        codes[r] = np.clip(n, -127, 127)
    return codes, scales


def product(a, sa, w, sw, bias=None):
    """Float32 results in the documented order; the sums exact in float64."""
    sums = a.astype(np.float64) @ w.astype(np.float64).T
    out = sums.astype(np.int64).astype(np.float32) * sa.astype(np.float32)[:, None] * sw.astype(np.float32)
    return out if bias is None else out + bias.astype(np.float32)


def log_probs(x, scale, tokens=None, n_top=0):
    """lse, entropy, ln p of the tokens, ids and ln p of the best, of float64 rows."""
    lse, entropy, lps, ids, tops = [], [], [], [], []
    for r, row in enumerate(x):
        bad = np.any(np.isnan(row)) or np.any(row == np.inf)
        z = row * np.float64(np.float32(scale))
        m = z.max() if not bad else 0.0
        if bad:
            p, total = np.full_like(z, np.nan), np.nan
        elif m == -np.inf:
            p, total = z, -np.inf
        else:
            more = np.log(np.exp(z - m).sum())
            total = m + more
            p = (z - m) - more  # far from 0, m would swallow it
        lse.append(total)
        if bad or m == -np.inf:
            entropy.append(np.nan if bad else 0.0)
        else:
            q = np.exp(p)
            entropy.append(-np.sum(np.where(q > 0, q * np.where(q > 0, p, 0), 0)))
        if tokens is not None:
            lps.append([0.0 if t == -1 else p[t] if 0 <= t < len(row) else np.nan for t in tokens[r]])
        key = np.where(np.isnan(row), -np.inf, row)
        order = np.lexsort((np.arange(len(row)), np.isnan(row), -key))[:n_top]
        ids.append(order)
        tops.append(p[order])
    return np.array(lse), np.array(entropy), np.array(lps), np.array(ids), np.array(tops)


def log_prob_bounds(x, scale, lse, entropy, lp):
    """Absolute bounds of (lse, entropy, ln p). A term 2^d: its exponent carries the factor's rounding
    and d's own (half a step each of the term's distance from the largest, at most 104 where it adds
    anything), the exponential one step, a thread's sum a half step an element (at most a 256th of the
    row and a turn's 32) and the joins some 40 more; the entropy's terms carry the same, times their d. lse
    carries half steps of the largest value's size, ln p of its own and of its distance."""
    top = np.max(np.where(np.isfinite(x), x, -np.inf)) if np.any(np.isfinite(x)) else 0.0
    span = min(104.0, max(0.0, (top - np.min(np.where(np.isfinite(x), x, top))) * scale)) + 1
    sums = (x.shape[-1] / 256 + 32 + 40) * U + 2 * U + 6 * span * U
    return (sums + 4 * U * (np.abs(lse) + abs(top) * scale), 3 * sums * (1 + span) + 4 * U * (1 + entropy), sums + 4 * U * (np.abs(lp) + span))
