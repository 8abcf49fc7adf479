"""NumPy oracles of the step plan and the block norm: the definitions, one request and one row at a
time, in whole numbers and in float64."""

import numpy as np

SEQ_RANGE, TABLE_SHORT, WORK_OVERFLOW, POOL_EMPTY = 4, 8, 16, 32
PAGE = 64


def step_plan(cached, new, table, free, count, tokens):
    """Returns ``(q_start, kv_len, seq_id, q_pos, slot, table, free_left, flags)``."""
    table = np.array(table, dtype=np.int64, copy=True)
    stack = list(np.asarray(free)[:max(0, min(int(count), len(free)))])
    columns, flags = table.shape[1], 0
    q_start, kv_len, rows = [0], [], []
    for s, (c, n) in enumerate(zip(cached, new)):
        c, n = int(c), int(n)
        if c < 0 or n < 0:
            flags |= SEQ_RANGE
        c, n = max(c, 0), max(n, 0)
        length = c + n
        first, last = -(-c // PAGE), -(-length // PAGE)
        if last > columns:
            flags |= TABLE_SHORT
            length = min(length, PAGE * columns)
        first, last = min(first, columns), min(last, columns)
        for col in range(first, last):
            if stack:
                table[s, col] = stack.pop()
            else:
                table[s, col] = -1
                flags |= POOL_EMPTY
                length = min(length, PAGE * min(col, last))
        kv_len.append(length)
        for p in range(c, c + n):
            col = p // PAGE
            page = table[s, col] if col < columns else -1
            rows.append((s, min(p, 2 ** 31 - 1), page * PAGE + p % PAGE if page >= 0 else -1))
        q_start.append(q_start[-1] + n)
    if q_start[-1] > tokens:
        flags |= WORK_OVERFLOW
    rows = rows[:tokens] + [(-1, -1, -1)] * (tokens - len(rows))
    seq_id, q_pos, slot = (np.array([r[i] for r in rows], dtype=np.int64) for i in range(3))
    return (np.minimum(q_start, tokens), np.array(kv_len, dtype=np.int64), seq_id, q_pos, slot, table,
            len(stack), flags)


def rms(v, eps):
    return v / np.sqrt((v * v).mean(axis=-1, keepdims=True) + eps)


def block_norm(y, residual, *, post_weight=None, gate=None, scale=1.0, pre_weight=None, eps=1e-6,
               post_eps=None):
    """``(out, x)`` in float64; ``x`` is None without ``pre_weight``."""
    y, residual = np.asarray(y, np.float64), np.asarray(residual, np.float64)
    b = y if post_weight is None else rms(y, eps if post_eps is None else post_eps) * post_weight
    if gate is not None:
        b = b * gate
    out = residual + scale * b
    return out, None if pre_weight is None else rms(out, eps) * pre_weight
