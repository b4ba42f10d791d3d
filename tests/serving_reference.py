"""Plain 64-bit restatements of the serving operators for their tests: numpy's
int64 (which wraps as the reference's sums do) and Python's integers for the
divisions. Every value has one right answer, so the tests compare for equality.
"""
import numpy as np

I32 = (-(2**31), 2**31 - 1)


def half_even(x, n):
    """x / 2^n rounded to nearest, ties to even (n > 0)."""
    f = x >> n
    rest = x - (f << n)
    half = np.int64(1) << (n - 1)
    return f + ((rest > half) | ((rest == half) & (f % 2 == 1)))


def score(sums, scale):
    """mistral.rs:130-145, or requantize where scale is 0."""
    if scale:
        # floor(sum * scale / 2^32), the sum in two halves
        hi, lo = sums >> 32, sums & 0xFFFFFFFF
        low = (lo.astype(np.uint64) * np.uint64(scale)) >> np.uint64(32)
        sums = hi * np.int64(scale) + low.astype(np.int64)
    return np.clip(half_even(sums, 16), *I32)


def exp_term(distance):
    """softmax_exp_term (ops.rs:508-556) of scores `distance` >= 0 below the maximum."""
    near = distance < 1 << 20
    x = np.where(near, distance, 0).astype(np.int64) << 16
    k, r = np.divmod(x, np.int64(2977044472))
    p2 = half_even(r * r, 32)
    p3 = half_even(p2 * r, 32)
    p4 = half_even(p3 * r, 32)
    p5 = half_even(p4 * r, 32)

    def over(p, n):
        a, b = np.divmod(p, n)
        return a + ((2 * b > n) | ((2 * b == n) & (a % 2 == 1)))

    e = (1 << 32) - r + over(p2, 2) - over(p3, 6) + over(p4, 24) - over(p5, 120)
    return np.where(near, np.where(k > 0, half_even(e, np.maximum(k, 1)), e), 0)


def weights(s):
    """attention_softmax (ops.rs:233-276) of one row of scores."""
    top = int(s.max())
    at = int((s == top).argmax())
    e = exp_term(np.minimum(top - s, 2**31 - 1))
    total = int(e.sum())
    w = np.zeros(len(e), np.int64)
    for i in np.nonzero(e)[0]:
        n, rest = divmod(int(e[i]) << 32, total)
        n += 2 * rest > total or (2 * rest == total and n % 2 == 1)
        w[i] = (n >> 16) + ((n & 0xFFFF) > 0x8000 or ((n & 0xFFFF) == 0x8000 and (n >> 16) % 2 == 1))
    w[at] += 65536 - int(w.sum())
    return w


def attend(q, k, v, scale):
    """One query [d] against keys and values [n][d] (all seen): int32 [d]."""
    if len(k) == 0:
        return np.zeros(len(q), np.int32)
    q, k, v = q.astype(np.int64), k.astype(np.int64), v.astype(np.int64)
    w = weights(score((k * q).sum(1), scale))
    return np.clip(half_even((w[:, None] * v).sum(0), 16), *I32).astype(np.int32)


def prompts(q, k, v, offsets, heads, kv_heads, scale, window):
    d = q.shape[1] // heads
    out = np.zeros(q.shape, np.int32)
    for a, b in zip(offsets[:-1], offsets[1:]):
        for i in range(a, b):
            lo = max(a, i + 1 - window) if window else a
            for h in range(heads):
                c = slice(h * d, (h + 1) * d)
                g = slice(h * kv_heads // heads * d, (h * kv_heads // heads + 1) * d)
                out[i, c] = attend(q[i, c], k[lo:i + 1, g], v[lo:i + 1, g], scale)
    return out


def trees(q, k_pages, v_pages, table, held, offsets, masks, positions, heads, kv_heads, scale, window):
    d = q.shape[1] // heads
    page, pool = k_pages.shape[1], k_pages.shape[0]
    out = np.zeros(q.shape, np.int32)
    for r, h0 in enumerate(held):
        a, b = offsets[r], offsets[r + 1]

        def row(t):
            c = t // page
            ok = c < table.shape[1] and 0 <= table[r, c] < pool
            return int(table[r, c]) * page + t % page if ok else -1

        for i in range(a, b):
            low = max(0, int(positions[i]) + 1 - window) if window else 0
            seen = [row(t) for t in range(low, h0)]
            seen += [row(h0 + j) for j in range(b - a)
                     if int(masks[i]) >> j & 1 and (not window or positions[a + j] >= low)]
            seen = [x for x in seen if x >= 0]
            for h in range(heads):
                c = slice(h * d, (h + 1) * d)
                g = slice(h * kv_heads // heads * d, (h * kv_heads // heads + 1) * d)
                kr = k_pages.reshape(-1, k_pages.shape[2])[seen][:, g]
                vr = v_pages.reshape(-1, v_pages.shape[2])[seen][:, g]
                out[i, c] = attend(q[i, c], kr, vr, scale)
    return out


def plan(held, fresh, table, free, page, tokens, parents=None):
    table = table.copy()
    offsets, slots, positions, masks = [0], [], [], []
    taken = 0
    for r, (h, f) in enumerate(zip(held, fresh)):
        for c in range(-(-h // page), -(-(h + f) // page)):
            if c < table.shape[1]:
                table[r, c] = free[taken] if taken < len(free) else -1
            taken += 1
        own = []
        for i in range(f):
            c = (h + i) // page
            p = int(table[r, c]) if c < table.shape[1] else -1
            slots.append(p * page + (h + i) % page if p >= 0 else -1)
            position = h + i
            if parents is not None:
                m, at, good = 0, i, i < 64
                while good:
                    m |= 1 << at
                    up = int(parents[offsets[-1] + at])
                    if up == -1:
                        break
                    good = 0 <= up < at
                    at = up
                own.append(m if good else 0)
                if good:
                    position = h + bin(m).count("1") - 1
            positions.append(position)
        masks += own
        offsets.append(offsets[-1] + f)
    pad = tokens - len(slots)
    if pad < 0:
        slots, positions, masks = slots[:tokens], positions[:tokens], masks[:tokens]
        pad = 0
    signed = np.array([m - (1 << 64) if m >> 63 else m for m in masks] + [0] * (pad if parents is not None else 0), np.int64)
    return (np.array(offsets, np.int32), np.array(slots + [-1] * pad, np.int64),
            np.array(positions + [0] * pad, np.int32), table, taken, signed)


def walk(parents, tokens, picks):
    """Accepted nodes of one request."""
    if len(parents) == 0:
        return []
    path = [0]
    while True:
        at = path[-1]
        below = [j for j in range(1, min(len(parents), 64)) if parents[j] == at < j and tokens[j] == picks[at]]
        if not below:
            return path
        path.append(below[0])
