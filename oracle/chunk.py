"""NumPy oracle of the chunk attention: one sequence, one head and one token block at a time, in
float64, from the definition (keys and values expanded per head, causal by position)."""

import numpy as np

from . import fp8

LATENT = 512


def pool_rows(pool, kv_format):
    """Pool rows ``u8 [P * 64, stride]`` as float64 values (FP8 rows: code times scale, unrounded)."""
    if kv_format == 1:
        return fp8.dequant_rows(pool)
    words = np.ascontiguousarray(pool[:, :1152 if kv_format == 2 else 1024]).view(np.uint16)
    return (words.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def chunk_attention(q, w_uk, w_uv, rows, page_table, q_start, q_pos, kv_len, *, scale, step=256):
    """``(out [T, H, Dv], lse [T, H])`` in float64; tokens of no sequence stay NaN.

    ``rows`` ``[P * 64, 512 + Dr]`` float64. Rows of pages outside the pool are zeros.
    """
    tokens, heads, _ = q.shape
    dn, dv = w_uk.shape[1], w_uv.shape[1]
    slots = page_table.shape[1]
    out = np.full((tokens, heads, dv), np.nan)
    lse = np.full((tokens, heads), np.nan)
    for s in range(len(kv_len)):
        b, e = int(q_start[s]), int(q_start[s + 1])
        n = max(0, min(int(kv_len[s]), 64 * slots))
        if e <= b:
            continue
        pos = np.arange(n)
        page = page_table[s][pos // 64].astype(np.int64)
        known = (page >= 0) & (page < len(rows) // 64)
        kv = np.where(known[:, None], rows[np.where(known, page, 0) * 64 + pos % 64], 0.0)
        good = np.isfinite(kv).all(axis=1)
        lat = np.where(good[:, None], kv, 0.0)
        seen = np.minimum(n, np.maximum(q_pos[b:e].astype(np.int64) + 1, 0))
        spoilt = np.array([not good[:m].all() for m in seen])
        for h in range(heads):
            k = np.concatenate([lat[:, :LATENT] @ w_uk[h].T, lat[:, LATENT:]], axis=1)
            v = lat[:, :LATENT] @ w_uv[h].T
            for a in range(b, e, step):
                z = min(e, a + step)
                score = scale * (q[a:z, h] @ k.T)
                score[pos[None] >= seen[a - b:z - b, None]] = -np.inf
                peak = score.max(axis=1, initial=-np.inf)
                p = np.exp(score - np.where(np.isinf(peak), 0.0, peak)[:, None])
                total = p.sum(axis=1)
                out[a:z, h] = (p @ v) / np.where(total > 0, total, 1.0)[:, None]
                with np.errstate(divide="ignore"):
                    lse[a:z, h] = np.where(total > 0, peak + np.log(total), -np.inf)
        out[b:e][spoilt] = np.nan
        lse[b:e][spoilt] = np.nan
    return out, lse
