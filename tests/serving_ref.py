"""Plain 64-bit restatements of the serving operators (include/litemind_serving.h) and the bounds their rounding allows."""
import numpy as np

STEP_ARRAYS = ("lengths", "starts", "positions", "slots", "queue", "info", "table", "ring")


def pages_of(tokens, page):
    return -(-int(tokens) // page)


def plan(cached, added, table, ring, queue, page, tokens, max_added):
    """lm_page_plan, a request and a token at a time.  Returns STEP_ARRAYS."""
    table, ring = table.copy(), ring.copy()
    R, width, pages = len(cached), table.shape[1], len(ring)
    head, count = int(queue[0]) % pages, int(queue[1])
    new = [max(int(a), 0) for a in added]
    status = 0
    if any(c < 0 or int(c) + n > width * page for c, n in zip(cached, new)):
        status = 1
    elif sum(new) > tokens or any(n > max_added for n in new):
        status = 2
    elif sum(pages_of(int(c) + n, page) - pages_of(c, page) for c, n in zip(cached, new)) > max(count, 0):
        status = 3
    out = {"table": table, "ring": ring, "positions": np.zeros(tokens, np.int32),
           "slots": np.full(tokens, -1, np.int32)}
    if status:
        return {**out, "lengths": np.asarray(cached, np.int32), "starts": np.zeros(R + 1, np.int32),
                "queue": np.array([head, count], np.int32), "info": np.array([status, 0, 0, 0], np.int32)}
    lengths, starts, taken, back = [], [0], 0, 0
    for r in range(R):
        c = int(cached[r])
        lengths.append(0 if added[r] < 0 else c + new[r])
        starts.append(starts[-1] + new[r])
        if added[r] < 0:
            for k in range(pages_of(c, page)):
                ring[(head + count + back) % pages] = table[r, k]
                back += 1
        held = pages_of(c, page)
        for i in range(new[r]):
            p = c + i
            if p // page >= held:
                table[r, held] = ring[(head + taken) % pages]
                held, taken = held + 1, taken + 1
            at, page_id = starts[r] + i, int(table[r, p // page])
            out["positions"][at] = p
            if 0 <= page_id < pages:
                out["slots"][at] = page_id * page + p % page
    return {**out, "lengths": np.array(lengths, np.int32), "starts": np.array(starts, np.int32),
            "queue": np.array([(head + taken) % pages, count - taken + back], np.int32),
            "info": np.array([0, starts[-1], taken, back], np.int32)}


def attention(q, rows, cached, scale, rank, unit):
    """One request: queries [n, heads, width] over its pool rows [cached + n, width], in 64 bits, and what the
    operator's roundings may add: `unit` the largest relative rounding of the 16-bit type.

    The weights e_j = exp(s_j - max) round to 16 bits, relative `unit` (below 2^-14 fp16 has a fixed step, off by at
    most 2^-25), the output once more.  A score's 32-bit sum of w products is off by at most (w + 2) 2^-24 of the sum
    of their magnitudes, times `scale`; that, the exponential's few units and the sums over n keys move a weight by a
    relative 2 ds + (n + 64) 2^-23.  An output channel is sum_j p_j c_j, so a weight's relative error e moves it by at
    most e sum_j p_j |c_j|, twice that with the total's own."""
    q, rows = q.astype(np.float64), rows.astype(np.float64)
    n, heads, width = q.shape
    out, bound = np.empty((n, heads, rank)), np.empty((n, heads, rank))
    for i in range(n):
        k = rows[:cached + i + 1]
        s = (q[i] @ k.T) * scale
        ds = (np.abs(q[i]) @ np.abs(k).T).max(1) * abs(scale) * (width + 2) * 2.0 ** -24
        e = np.exp(s - s.max(1, keepdims=True))
        total = e.sum(1, keepdims=True)
        c = np.abs(k[:, :rank])
        out[i] = (e / total) @ k[:, :rank]
        spread = (e / total) @ c
        other = (2 * ds + (len(k) + 64) * 2.0 ** -23)[:, None]
        bound[i] = spread * (unit + 2 * other) + c.sum(0) * 2.0 ** -25 / total + np.abs(out[i]) * unit + 2.0 ** -24
    return out, bound


def sample(logits, temperature, top_k, top_p, min_p, u):
    """One row: (token, probability, how near u lies to the border of another token, relative to the total)."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, np.inf
    if not temperature > 0:
        return int(np.argmax(x)), 1.0, np.inf
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    with np.errstate(invalid="ignore"):
        e = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(temperature)))
    if top == np.inf:
        e = (x[order] == np.inf).astype(np.float64)
    keep = min(int(top_k), len(order)) if top_k > 0 else len(order)
    near = np.inf
    if top_p < 1:
        before = np.cumsum(e[:keep]) - e[:keep]
        total = e[:keep].sum()
        # the first token is kept whatever the sums
        near = np.abs(before[1:] - top_p * total).min(initial=np.inf) / total if top_p > 0 else np.inf
        keep = max(1, int((before < top_p * total).sum()))
    if min_p > 0:
        # the largest logit's e is 1 on every side
        near = min(near, np.abs(e[:keep][e[:keep] != 1.0] - np.float64(min_p)).min(initial=np.inf))
        keep = max(1, min(keep, int((e[:keep] >= np.float64(min_p)).sum())))
    at = np.sort(order[:keep])
    inverse = np.empty(len(x))
    inverse[order] = e
    w = inverse[at]
    running = np.cumsum(w)
    target = np.float64(u) * running[-1]
    k = min(int((running <= target).sum()), int(np.flatnonzero(w > 0)[-1]))
    near = min(near, np.abs(running - target).min() / running[-1])
    return int(at[k]), float(w[k] / running[-1]), float(near)
