"""float64 / integer oracles of the paged-cache operators, request by request and token by token (NumPy)."""
import numpy as np

from .afa_oracle import octic


def plan(table, held, lens, new, stack, free, page, max_tokens, parents=None):
    """The step ``paged_plan`` describes, one request after the other. Arrays are not modified."""
    table, stack = np.array(table), np.array(stack)
    batch, cols = table.shape
    state = [int(x) for x in stack[:int(free)]]
    lens, new = np.maximum(lens, 0).astype(int), np.maximum(new, 0).astype(int)
    want = lens + new
    need = -(-want // page)
    refused = np.zeros(batch, bool)
    asked = 0
    for b in range(batch):
        if want[b] > cols * page or (parents is not None and new[b] > parents.shape[1]):
            refused[b] = True
            continue
        asked += new[b]
        refused[b] = new[b] > 0 and asked > max_tokens
    for b in range(batch):  # released pages, in request order
        if not refused[b]:
            state += [int(x) for x in table[b, need[b]:max(need[b], held[b])]]
    supply, grown = len(state), 0
    for b in range(batch):
        grow = 0 if refused[b] else max(0, need[b] - held[b])
        grown += grow
        if grow and grown > supply:
            refused[b] = True
            continue
        for j in range(grow):
            table[b, held[b] + j] = state.pop()
    state = state[:len(stack)]  # released pages that find no room are lost
    if len(state) > free:
        stack[int(free):len(state)] = state[int(free):]
    slots, rows, positions, words = [], [], [], []
    cu = [0]
    nwords = 0 if parents is None else -(-parents.shape[1] // 32)
    for b in range(batch):
        n = 0 if refused[b] else new[b]
        cu.append(cu[-1] + n)
        for i in range(n):
            at = lens[b] + i
            slots.append(int(table[b, at // page]) * page + at % page)
            rows.append(b)
            depth = i
            if parents is not None:
                depth, node, bits = 0, i, 1 << i
                while 0 <= parents[b, node] < node:
                    node = int(parents[b, node])
                    bits |= 1 << node
                    depth += 1
                words.append([(bits >> (32 * w)) & 0xFFFFFFFF for w in range(nwords)])
            positions.append(lens[b] + depth)
    behind = max_tokens - len(slots)
    out = {
        "slots": np.array(slots + [-1] * behind, np.int64), "rows": np.array(rows + [-1] * behind, np.int32),
        "positions": np.array(positions + [0] * behind, np.int32), "cu_tokens": np.array(cu, np.int32),
        "seq_lens": np.where(refused, lens, want).astype(np.int32),
        "page_counts": np.where(refused, held, need).astype(np.int32), "free_count": np.array([len(state)], np.int32),
        "granted": ~refused, "block_table": table, "free_pages": stack}
    if parents is not None:
        out["ancestors"] = np.array(words + [[0] * nwords] * behind, np.uint32).reshape(max_tokens, nwords)
    return out


def rotate_axes(x, c, s, positions, sections, back=False):
    """x (..., heads, tokens, dim) with positions (axes, ..., tokens)."""
    y = np.array(x, np.float64)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    for p, a in enumerate(axis):
        cc, ss = (np.asarray(t, np.float64)[np.asarray(positions[a]), p][..., None, :] for t in (c, s))
        ss = -ss if back else ss
        x0, x1 = np.asarray(x, np.float64)[..., 2 * p], np.asarray(x, np.float64)[..., 2 * p + 1]
        y[..., 2 * p], y[..., 2 * p + 1] = cc * x0 - ss * x1, ss * x0 + cc * x1
    return y


def attend(q, k_cache, v_cache, table, lens, cu, ancestors=None, sink=0.5):
    """(out, d_total) float64; rows of no request are NaN."""
    tokens, heads, dim = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    out, den = np.full(q.shape, np.nan), np.full((tokens, heads), np.nan)
    for b in range(len(lens)):
        n, length = int(cu[b + 1] - cu[b]), int(lens[b])
        held = [int(table[b, j // page]) for j in range(length)]
        ok = np.array([0 <= p < pages for p in held], bool)
        rows = [(p if g else 0, j % page) for j, (p, g) in enumerate(zip(held, ok))]
        k, v = (np.array([x[p, :, r] for p, r in rows], np.float64).reshape(length, kv_heads, dim)
                for x in (k_cache, v_cache))
        for i in range(n):
            seen = np.zeros(length, bool)
            for j in range(length):
                node = j - (length - n)
                if ancestors is None:
                    seen[j] = node <= i
                else:
                    w = node >> 5
                    seen[j] = node < 0 or (w < ancestors.shape[1] and
                                           (int(ancestors[cu[b] + i, w]) >> (node & 31)) & 1)
            seen &= ok
            for h in range(heads):
                g = h // (heads // kv_heads)
                p = octic(k[seen, g] @ np.asarray(q[cu[b] + i, h], np.float64) / np.sqrt(dim))
                d = p.sum() + sink
                den[cu[b] + i, h] = d
                out[cu[b] + i, h] = p @ v[seen, g] / d if d > 0 else 0.0
    return out, den


def commit(k_cache, v_cache, table, base, lens, accepted):
    """(lens, k_cache, v_cache) after the moves; caches (layers, pages, heads, page, dim)."""
    k_cache, v_cache = np.array(k_cache), np.array(v_cache)
    pages, page = k_cache.shape[1], k_cache.shape[3]
    out = []
    for b, path in enumerate(accepted):
        last, count = -1, 0
        for i, node in enumerate(path):
            src, dst = base[b] + node, base[b] + i
            if node <= last or src >= min(lens[b], table.shape[1] * page):
                break
            ps, pd = table[b, src // page], table[b, dst // page]
            if not (0 <= ps < pages and 0 <= pd < pages):
                break
            for x in (k_cache, v_cache):
                x[:, pd, :, dst % page] = x[:, ps, :, src % page]
            last, count = node, count + 1
        out.append(max(base[b], 0) + count)
    return np.array(out, np.int32), k_cache, v_cache
