"""Oracle of the index branch (write, scores, select) in float64 NumPy, from the definitions in
``include/tq_mla.h``. No counterpart in the reference, whose contract takes selected indices as
given (crates/tq-core/src/contracts.rs:196-200)."""

import numpy as np

from . import fp8

PAGE = 64
DIM = 128


def turned(x, pos, freq, start, half, mscale=1.0):
    """Rows ``[T, ..., 128]`` with ``2 len(freq)`` values from ``start`` on turned by their position."""
    x = np.array(x, dtype=np.float64)
    n = len(freq)
    i = np.arange(n)
    re, im = (start + i, start + i + n) if half else (start + 2 * i, start + 2 * i + 1)
    angle = np.asarray(pos, dtype=np.float64)[:, None] * np.asarray(freq, dtype=np.float64)
    angle = angle.reshape((len(angle),) + (1,) * (x.ndim - 2) + (n,))
    a, b = x[..., re].copy(), x[..., im].copy()
    x[..., re] = mscale * (a * np.cos(angle) - b * np.sin(angle))
    x[..., im] = mscale * (a * np.sin(angle) + b * np.cos(angle))
    return x


def normalised(k, weight, bias, eps):
    k = np.asarray(k, dtype=np.float64)
    if bias is not None:
        k = k - k.mean(axis=1, keepdims=True)
    k = k / np.sqrt((k * k).mean(axis=1, keepdims=True) + eps) * weight
    return k if bias is None else k + bias


def slots(page_table, seq_id, pos, pages):
    """Pool row of each token, -1 where it has none, and the flags of those."""
    rows, flags = np.full(len(pos), -1, dtype=np.int64), 0
    for t, (s, p) in enumerate(zip(seq_id, pos)):
        if not 0 <= s < page_table.shape[0]:
            flags |= 4
        elif p < 0 or p // PAGE >= page_table.shape[1]:
            flags |= 8
        elif not 0 <= page_table[s, p // PAGE] < pages:
            flags |= 2
        else:
            rows[t] = int(page_table[s, p // PAGE]) * PAGE + p % PAGE
    return rows, flags


def sees(seq_id, q_pos, kv_len, most):
    n = [min(int(kv_len[s]), int(p) + 1) if 0 <= s < len(kv_len) else 0 for s, p in zip(seq_id, q_pos)]
    return np.clip(n, 0, most)


def codes_value(codes):
    return fp8.e4m3_table()[np.asarray(codes, dtype=np.uint8)]


def scores(q_codes, w, rows, page_table, seq_id, q_pos, kv_len, columns, fill):
    """``rows`` u8 ``[P * 64, r]``. Returns the scores (``fill`` where nothing is seen) and, for
    bounds, the same sums over the magnitudes of all products."""
    t, h, _ = q_codes.shape
    out, mass = np.array(fill, dtype=np.float64), np.zeros((t, columns))
    q = codes_value(q_codes)
    key = codes_value(rows[:, :DIM])
    scale = np.ascontiguousarray(rows[:, DIM:DIM + 4]).view(np.float32)[:, 0].astype(np.float64)
    pages = len(rows) // PAGE
    n_all = sees(seq_id, q_pos, kv_len, min(columns, PAGE * page_table.shape[1]))
    for i in range(t):
        n = int(n_all[i])
        if n == 0:
            continue
        page = page_table[seq_id[i], np.arange(n) // PAGE].astype(np.int64)
        known = (page >= 0) & (page < pages)
        at = np.where(known, page, 0) * PAGE + np.arange(n) % PAGE
        k = np.where(known[:, None], key[at], 0.0)
        s = np.where(known, scale[at], 0.0)
        with np.errstate(invalid="ignore"):
            dots = k @ q[i].T
            out[i, :n] = s * (np.where(dots < 0, 0.0, dots) @ np.asarray(w[i], dtype=np.float64))
            mass[i, :n] = np.abs(s) * ((np.abs(k) @ np.abs(q[i]).T) @ np.abs(np.asarray(w[i], dtype=np.float64)))
    return out, mass


def select(score, seq_id, q_pos, kv_len, k, page_table=None, keep_first=0, keep_last=0):
    t, columns = score.shape
    idx, length = np.full((t, k), -1, dtype=np.int64), np.zeros(t, dtype=np.int64)
    most = columns if page_table is None else min(columns, PAGE * page_table.shape[1])
    for i, n in enumerate(sees(seq_id, q_pos, kv_len, most)):
        if n == 0:
            continue
        v = np.where(np.isnan(score[i, :n]), -np.inf, score[i, :n].astype(np.float64))
        if page_table is not None:
            v = np.array([v[j:j + PAGE].max() for j in range(0, n, PAGE)])
        m = len(v)
        place = np.arange(m)
        kept = (place < keep_first) | (place >= m - keep_last)
        order = np.lexsort((place, -v, ~kept))
        order = [j for j in order if kept[j] or v[j] > -np.inf][:k]
        best = np.sort(np.array(order, dtype=np.int64))
        length[i] = len(best)
        if page_table is not None:
            length[i] = sum(min(PAGE, n - PAGE * j) for j in best)
            best = page_table[seq_id[i], best]
        idx[i, :len(best)] = best
    return idx, length
