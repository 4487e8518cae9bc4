"""Plain 64-bit implementations of the cache operators, row by row in numpy, for the tests.

Caches are numpy arrays: K uint32 [pool, W], V uint8 [pool, D]; cache row r's slot t lives
in pool row table[r, t // block] * block + t % block, or r * cap + t without a table."""
import numpy as np
import torch

FP8 = torch.float8_e4m3fn


def place(table, block, nb, r, t):
    page = int(table[r, t // block]) if table is not None else r * nb + t // block
    return page * block + t % block


def make_table(rows, nb, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(rows * nb, generator=g).to(torch.int32).view(rows, nb)


def words(up):
    """Sign words of a boolean [..., D]."""
    up = np.asarray(up).reshape(*up.shape[:-1], up.shape[-1] // 32, 32).astype(np.uint64)
    return (up << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def rotate(x, table_row, layout):
    """x float64 [D] turned by a table row float64 [2, rot / 2]; every product is exact."""
    out = x.copy()
    c, s = table_row
    h = c.size
    i, j = (np.arange(h), np.arange(h) + h) if layout == "half" else (2 * np.arange(h), 2 * np.arange(h) + 1)
    with np.errstate(invalid="ignore", over="ignore"):
        out[i] = x[i] * c - x[j] * s
        out[j] = x[j] * c + x[i] * s
    return out


def codes(v, scale):
    """e4m3 codes of clamp(v / scale, -448, 448) by torch: v, scale float32 tensors."""
    return (v.float() / scale).clamp(-448.0, 448.0).to(FP8).view(torch.uint8).numpy()


def key_weights(q, k_cache, ctx, table, block, nb, seq_q, inv, causal, group, q_first, n_q, decay, w):
    """[rows, ld] float64; entries at or beyond the length stay as in w."""
    out = np.asarray(w, dtype=np.float64).copy()
    pool_blocks = k_cache.shape[0] // block
    D = 32 * q.shape[1]
    for r, n in enumerate(ctx):
        n = max(0, min(int(n), block * nb))
        at = [(place(table, block, nb, r, t), table is None or 0 <= int(table[r, t // block]) < pool_blocks) for t in range(n)]
        good = np.array([ok for _, ok in at], dtype=bool)
        rows = np.array([p if ok else 0 for p, ok in at], dtype=np.int64)
        total = np.zeros(n)
        first = 0 if q_first is None else int(q_first[r])
        for g in range(group):
            for i in range(first, first + n_q):
                if not 0 <= i < seq_q or n == 0:
                    continue
                seen = good & (np.arange(n) <= i) if causal else good
                if not seen.any():
                    continue
                x = q[(r * group + g) * seq_q + i][None] ^ k_cache[rows]
                pop = np.unpackbits(x.view(np.uint8), axis=1).sum(1)
                s = (D - 2.0 * pop) * float(np.float32(inv))
                e = np.where(seen, np.exp(np.maximum(s - s[seen].max(), -80.0)), 0.0)
                total += e / e.sum()
        out[r, :n] = float(np.float32(decay)) * out[r, :n] + total
    return out


def key_weights_tolerance(n, rows, inv, D):
    """Relative: an exponential of an argument rounded to f32 (at most 80), a table or
    hardware exponential (64 half steps cover 2^-19), and f32 sums of positive terms over
    at most n / 128 keys a thread and `rows` queries."""
    return 2.0**-24 * (n / 128 + rows + 64 + 2 * min(80.0, 2 * abs(inv) * D))


def evict(k, v, scale, ctx, table, block, nb, w, pos, keep, sink, recent):
    """Returns (k, v, scale, ctx, w, pos) after the eviction; the inputs stay."""
    k, v, w, pos = k.copy(), v.copy(), w.copy(), pos.copy()
    scale = None if scale is None else scale.copy()
    new = np.zeros(len(ctx), dtype=np.int32)
    pool_blocks = k.shape[0] // block
    for r, n in enumerate(ctx):
        n = max(0, min(int(n), block * nb))
        m = min(n, max(0, int(keep if np.isscalar(keep) else keep[r])))
        new[r] = m
        if m == n:
            continue
        p, x = pos[r, :n].astype(np.int64), w[r, :n]
        guard = (p < sink) | (p > p.max() - recent)
        # descending: protected, numbers, NaN; equal ones by slot
        klass = np.where(guard, 2, np.where(np.isnan(x), 0, 1))
        value = np.where(klass == 1, x, 0.0)
        order = np.lexsort((np.arange(n), -value, -klass))
        kept = np.zeros(n, dtype=bool)
        kept[order[:m]] = True
        empty, late = np.flatnonzero(~kept[:m]), m + np.flatnonzero(kept[m:])
        assert empty.size == late.size
        for dst, src in zip(empty, late):
            w[r, dst], pos[r, dst] = w[r, src], pos[r, src]
            pages = [0, 0] if table is None else [int(table[r, t // block]) for t in (dst, src)]
            if all(0 <= q < pool_blocks for q in pages):
                a, b = place(table, block, nb, r, dst), place(table, block, nb, r, src)
                k[a], v[a] = k[b], v[b]
                if scale is not None:
                    scale[a] = scale[b]
        w[r, m:n], pos[r, m:n] = 0.0, -1
    return k, v, scale, new, w, pos
