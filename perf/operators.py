"""The paged-cache operators as cases: what each is given, its plain form and its value in 64 bits.

A serving step with drafted tokens runs them in this order: ``paged_plan`` (block tables, slot maps and tree
masks from request lengths), ``paged_append`` (several-axis rotary of q and k, k and v into the cache),
``afa_paged`` (octic attention of the new tokens over the cache) and ``paged_commit`` (the accepted path of a
tree moves to the front). ``apply_ago_rotations_axes`` is the rotary alone, with its gradient, for training.

Caches are (pages, kv_heads, page_size, dim); queries (tokens, heads, dim), the requests' tokens one after the
other.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SINK = 0.5


# ----------------------------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # The smallest step: eight requests append one token each. Launch latency.
        {"name": "plan-decode", "op": "plan", "batch": 8, "page": 16, "new": 1, "nodes": 0, "length": 900,
         "short": False},
        # A full batch of drafted trees, with requests that ended since the last step.
        {"name": "plan-tree", "op": "plan", "batch": 256, "page": 32, "new": 48, "nodes": 64, "length": 8192,
         "short": False},
        # Training: queries and keys of a batch of image and text tokens, three axes, forward and backward.
        {"name": "rotate-train", "op": "rotate", "batch": 2, "heads": 32, "kv_heads": 8, "tokens": 4096, "dim": 128,
         "sections": "16,24,24", "span": 4096, "dtype": "bf16"},
        # A short odd sequence in float32, two axes, part of the channels left as they are.
        {"name": "rotate-odd", "op": "rotate", "batch": 1, "heads": 5, "kv_heads": 1, "tokens": 777, "dim": 64,
         "sections": "11,9", "span": 300, "dtype": "f32"},
        # Drafted trees of 64 requests into the cache.
        {"name": "append-tree", "op": "append", "tokens": 1536, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "sections": "16,24,24", "span": 8192, "dtype": "bf16"},
        # One token for each of seven requests.
        {"name": "append-decode", "op": "append", "tokens": 7, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "sections": "64", "span": 2048, "dtype": "bf16"},
        # The benchmark's decode batch over a paged cache, four query heads to a key head: the cache is what is read.
        {"name": "attend-decode", "op": "attend", "batch": 64, "new": 1, "length": 8192, "kv_heads": 8, "group": 4,
         "dim": 128, "page": 32, "tree": False, "dtype": "bf16"},
        # Trees of up to 48 drafted nodes after prompts of a few thousand tokens.
        {"name": "attend-tree", "op": "attend", "batch": 16, "new": 48, "length": 6000, "kv_heads": 8, "group": 4,
         "dim": 128, "page": 16, "tree": True, "dtype": "bf16"},
        # Chunks of long prompts, causal: tensor-core work.
        {"name": "attend-chunk", "op": "attend", "batch": 2, "new": 2048, "length": 8192, "kv_heads": 8, "group": 4,
         "dim": 128, "page": 128, "tree": False, "dtype": "bf16"},
        # A few short requests in float32.
        {"name": "attend-f32", "op": "attend", "batch": 5, "new": 7, "length": 1300, "kv_heads": 3, "group": 5,
         "dim": 64, "page": 16, "tree": True, "dtype": "f32"},
        # The accepted paths of 64 trees, eight layers' caches at once.
        {"name": "commit", "op": "commit", "batch": 64, "layers": 8, "kv_heads": 8, "dim": 128, "page": 32,
         "nodes": 48, "path": 8, "length": 300, "dtype": "bf16"},
        # The accepted paths of three small trees in one layer.
        {"name": "commit-small", "op": "commit", "batch": 3, "layers": 1, "kv_heads": 2, "dim": 64, "page": 16,
         "nodes": 21, "path": 5, "length": 100, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rotate", "append", "attend", "attend", "attend", "commit"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "plan":
        nodes = rng.choice([0, rng.randint(1, 128)])
        new = rng.randint(1, nodes) if nodes else _log(rng, 1, 1000)
        batch = _log(rng, 1, 256)
        return {"op": op, "batch": batch, "page": page, "new": min(new, max(1, 16000 // batch)), "nodes": nodes,
                "length": _log(rng, 1, 8192), "short": rng.random() < 0.3}
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "attend":
        tree = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        length = _log(rng, 1, 16384)
        new = min(length, rng.randint(1, 100) if tree else rng.choice([1, 1, _log(rng, 1, 2048)]))
        scores = 1.0e9 if dtype == "bf16" else 1.0e8
        new = max(1, min(new, int(scores / (group * kv_heads * length))))
        most = min(64 * 8192 * 8 // (length * kv_heads), int(scores / (new * group * kv_heads * length)))
        return {"op": op, "batch": _log(rng, 1, max(1, min(64, most))), "new": new, "length": length,
                "kv_heads": kv_heads, "group": group, "dim": dim, "page": page, "tree": tree, "dtype": dtype}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "commit":
        nodes = rng.randint(1, 64)
        return {"op": op, "batch": _log(rng, 1, 64), "layers": rng.randint(1, 8), "kv_heads": kv_heads, "dim": dim,
                "page": page, "nodes": nodes, "path": rng.randint(1, min(nodes, 12)), "length": rng.randint(1, 300),
                "dtype": dtype}
    axes = rng.randint(1, 3)
    left, sections = dim // 2, []
    for a in range(axes):
        sections.append(rng.randint(1, left - (axes - 1 - a)))
        left -= sections[-1]
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "sections": ",".join(map(str, sections)), "span": _log(rng, 16, 8192), "dtype": dtype}
    if op == "rotate":
        return {**case, "batch": rng.randint(1, 2), "tokens": _log(rng, 1, 4096)}
    return {**case, "tokens": _log(rng, 1, 4096), "page": page}


# ----------------------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------------------
def _up(a, b):
    return -(-a // b)


def _dev(x, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(x))
    return t.to(device="cuda", dtype=dtype or t.dtype)


def _tree(rng, n):
    """Parents of a drafted tree of n nodes, -1 for a root; mostly long branches."""
    back = np.minimum(rng.geometric(0.4, n), np.arange(n) + 1)
    return np.arange(n) - back


def _ancestors(parents):
    """Whether node j lies on node i's path to its root, and each node's depth."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        if 0 <= parents[i] < i:
            seen[i] = seen[parents[i]]
        seen[i, i] = True
    return seen, seen.sum(1) - 1


def _words(seen, count):
    full = np.zeros((seen.shape[0], 32 * count), np.uint32)
    full[:, : seen.shape[1]] = seen
    return (full.reshape(seen.shape[0], count, 32) << np.arange(32, dtype=np.uint32)).sum(2).astype(np.uint32).view(
        np.int32)


def _ragged(rng, batch, most):
    n = rng.integers(max(1, most // 2), most + 1, batch)
    n[rng.integers(batch)] = most
    return n


def _sizes(case):
    """Each request's new tokens and its length with them: the same for every seed, so that outputs keep their
    shapes."""
    rng = np.random.default_rng(case["batch"] + 1000 * case["length"])
    new = _ragged(rng, case["batch"], case["new"])
    return new, np.maximum(_ragged(rng, case["batch"], case["length"]), new)


def _tables(dim, span):
    """Rotation tables (span, dim / 2) of the rational frequencies, from their angles in 64 bits."""
    pairs = dim // 2
    w = 1.0 / (1.0 + (math.sqrt(10000.0) - 1.0) / max(pairs - 1, 1) * np.arange(pairs)) ** 2
    angle = np.arange(span)[:, None] * (2.0 * np.arctan(w))[None]
    return np.cos(angle), np.sin(angle)


def _sections(case):
    return tuple(int(x) for x in case["sections"].split(","))


def _pool(rng, lengths, page, columns):
    """A block table of shuffled pages that holds `lengths` tokens; the entries behind are -1."""
    held = -(-lengths // page)
    order = rng.permutation(int(held.sum()))
    table = np.full((len(lengths), columns), -1, np.int32)
    inside = np.arange(columns)[None] < held[:, None]
    table[inside] = order
    return table, len(order)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES.get(case.get("dtype"), torch.float32)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "plan":
        batch, page = case["batch"], case["page"]
        lens = rng.integers(0, case["length"] + 1, batch)
        lens[rng.random(batch) < 0.1] = 0  # ended since the last step
        held = -(-(lens + rng.integers(0, 3 * page, batch)) // page)
        new = _ragged(rng, batch, case["new"])
        new[lens == 0] = rng.integers(0, 2, int((lens == 0).sum())) * new[lens == 0]
        columns = _up(case["length"] + 3 * page + case["new"], page)
        order = rng.permutation(batch * columns)
        table = np.full((batch, columns), -1, np.int32)
        table[np.arange(columns)[None] < held[:, None]] = order[: int(held.sum())]
        rest = order[int(held.sum()):]
        stack = np.zeros(len(order), np.int32)
        stack[: len(rest)] = rest
        s.update(table=_dev(table), held=_dev(held, torch.int32), lens=_dev(lens, torch.int32),
                 new=_dev(new, torch.int32), stack=_dev(stack),
                 free=_dev(np.array([len(rest) // 8 if case["short"] else len(rest)], np.int32)),
                 max_tokens=batch * case["new"], parents=None)
        if case["nodes"]:
            s["parents"] = _dev(np.stack([_tree(rng, case["nodes"]) for _ in range(batch)]), torch.int32)
        return s
    if case["op"] in ("rotate", "append"):
        c, sn = _tables(case["dim"], case["span"])
        axes = len(_sections(case))
        s.update(c=_dev(c, torch.float32), s=_dev(sn, torch.float32), sections=_sections(case))
        if case["op"] == "rotate":
            b, t, d = case["batch"], case["tokens"], case["dim"]
            s["positions"] = _dev(rng.integers(0, case["span"], (axes, b, t)), torch.int32)
            s.update(q=randn(b, case["heads"], t, d), k=randn(b, case["kv_heads"], t, d),
                     gq=randn(b, case["heads"], t, d), gk=randn(b, case["kv_heads"], t, d))
            return s
        t, d, page = case["tokens"], case["dim"], case["page"]
        s["positions"] = _dev(rng.integers(0, case["span"], (axes, t)), torch.int32)
        pages = _up(t, page) + 3
        s.update(q=randn(t, case["heads"], d), k=randn(t, case["kv_heads"], d), v=randn(t, case["kv_heads"], d),
                 k_cache=randn(pages, case["kv_heads"], page, d), v_cache=randn(pages, case["kv_heads"], page, d),
                 slots=_dev(rng.permutation(pages * page)[:t]))
        return s
    if case["op"] == "commit":
        batch, page, d, h = case["batch"], case["page"], case["dim"], case["kv_heads"]
        base = np.random.default_rng(batch).integers(0, case["length"] + 1, batch)
        table, pages = _pool(rng, base + case["nodes"], page, _up(case["length"] + case["nodes"], page))
        count = rng.integers(1, case["path"] + 1, batch)
        accepted = np.full((batch, case["path"]), -1, np.int32)
        for b in range(batch):
            accepted[b, : count[b]] = np.sort(rng.permutation(case["nodes"])[: count[b]])
        s.update(k_cache=randn(case["layers"], pages, h, page, d), v_cache=randn(case["layers"], pages, h, page, d),
                 table=_dev(table), base=_dev(base, torch.int32), lens=_dev(base + case["nodes"], torch.int32),
                 accepted=_dev(accepted))
        return s
    batch, page, d, h, g = case["batch"], case["page"], case["dim"], case["kv_heads"], case["group"]
    new, lens = _sizes(case)
    cu = np.concatenate([[0], np.cumsum(new)])
    total = int(cu[-1])
    table, pages = _pool(rng, lens, page, _up(int(lens.max()), page))
    s.update(q=randn(total, h * g, d), k_cache=randn(pages, h, page, d), v_cache=randn(pages, h, page, d),
             table=_dev(table), lens=_dev(lens, torch.int32), cu=_dev(cu, torch.int32),
             rows=_dev(np.repeat(np.arange(batch), new)),
             node=_dev(np.arange(total) - np.repeat(cu[:-1], new)), most=int(new.max()), longest=int(lens.max()),
             ancestors=None)
    if case["tree"]:
        count = _up(case["new"], 32)
        s["ancestors"] = _dev(np.concatenate([_words(_ancestors(_tree(rng, n))[0], count) for n in new]))
    return s


# ----------------------------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------------------------
def _bits(words):
    """int32 words -> truth values, bit 0 first."""
    at = torch.arange(32, device=words.device)
    return (((words.long() & 0xFFFFFFFF)[..., None] >> at) & 1).bool().flatten(-2)


def _closure(parents):
    """(batch, n, n): whether j lies on i's path to its root (i itself among it)."""
    n = parents.shape[-1]
    at = torch.arange(n, device=parents.device)
    step = (parents[..., None] == at) & (at < at[:, None])
    reach = (step | torch.eye(n, dtype=torch.bool, device=parents.device)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (reach @ reach > 0).float()
    return reach.bool()


def _plan(s):
    table, page, cap = s["table"].long(), s["case"]["page"], s["max_tokens"]
    batch, columns = table.shape
    dev = table.device
    lens, new, fc = s["lens"].long().clamp(min=0), s["new"].long().clamp(min=0), s["free"].long()
    held = s["held"].long().clamp(0, columns)
    want = lens + new
    need = (want + page - 1) // page
    off = want > columns * page
    if s["parents"] is not None:
        off = off | (new > s["parents"].shape[1])
    ask = torch.where(off, 0, new)
    off = off | ((ask > 0) & (ask.cumsum(0) > cap))
    drop = torch.where(off, 0, (held - need).clamp(min=0))
    grow = torch.where(off, 0, (need - held).clamp(min=0))
    dropped = drop.sum()
    granted = ~(off | ((grow > 0) & (grow.cumsum(0) > fc + dropped)))
    grown = torch.where(granted, grow, 0)
    taken = grown.sum()
    n = torch.where(granted, new, 0)
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    at = torch.arange(columns, device=dev)[None]
    # released pages, request by request, behind the stack
    room = table.new_zeros(batch * columns + 1)
    gone = (at >= need[:, None]) & (at < (need + drop)[:, None])
    room[torch.where(gone, (drop.cumsum(0) - drop - need)[:, None] + at, batch * columns)] = table
    stack = s["stack"].long()
    place = torch.arange(len(stack), device=dev)

    def of_stack(i):
        i = i.clamp(min=0)
        return torch.where(i < fc, stack[i.clamp(max=len(stack) - 1)], room[(i - fc).clamp(0, batch * columns)])

    come = (at >= held[:, None]) & (at < (held + grown)[:, None])
    table = torch.where(come, of_stack(fc + dropped - 1 - ((grow.cumsum(0) - grow - held)[:, None] + at)), table)
    stack = torch.where((place >= fc) & (place < fc + dropped - taken), of_stack(place), stack)
    t = torch.arange(cap, device=dev)
    live = t < cu[-1]
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=batch - 1)
    node = t - cu[row]
    pos = lens[row] + node
    slots = torch.where(live, table[row, (pos // page).clamp(0, columns - 1)] * page + pos % page, -1)
    words = None
    if s["parents"] is not None:
        nodes = s["parents"].shape[1]
        seen = _closure(s["parents"].long())[row, node.clamp(0, nodes - 1)] & live[:, None]
        pos = lens[row] + seen.sum(1) - 1
        count = _up(nodes, 32)
        seen = torch.nn.functional.pad(seen, (0, 32 * count - nodes)).unflatten(1, (count, 32)).long()
        words = (seen << torch.arange(32, device=dev)).sum(2).to(torch.int32)
    s["table"].copy_(table)
    s["stack"].copy_(stack)
    return {"slots": slots, "rows": torch.where(live, row, -1).to(torch.int32),
            "positions": torch.where(live, pos, 0).to(torch.int32), "cu_tokens": cu.to(torch.int32),
            "seq_lens": torch.where(granted, want, lens).to(torch.int32),
            "page_counts": torch.where(granted, need, held).to(torch.int32),
            "free_count": (fc + dropped - taken).to(torch.int32), "granted": granted, "ancestors": words,
            "block_table": s["table"], "free_pages": s["stack"]}


def _factors(s, dim):
    """The tables' rows at each token's positions, (..., tokens, dim / 2); 1 and 0 where no axis turns a pair."""
    pos, pairs = s["positions"].long(), dim // 2
    parts = list(s["sections"])
    axis = torch.repeat_interleave(torch.arange(len(parts)), torch.tensor(parts)).tolist()
    pair = torch.arange(len(axis), device=pos.device)
    at = pos[axis].movedim(0, -1)
    pad = (0, pairs - len(axis))
    return (torch.nn.functional.pad(s["c"][at, pair], pad, value=1.0),
            torch.nn.functional.pad(s["s"][at, pair], pad, value=0.0))


def _turn(x, c, s):
    x0, x1 = x.float()[..., 0::2], x.float()[..., 1::2]
    return torch.stack([c * x0 - s * x1, s * x0 + c * x1], -1).flatten(-2).to(x.dtype)


def _rotate(s):
    c, sn = (f[:, None] for f in _factors(s, s["q"].shape[-1]))
    return {"q": _turn(s["q"], c, sn), "k": _turn(s["k"], c, sn), "dq": _turn(s["gq"], c, -sn),
            "dk": _turn(s["gk"], c, -sn)}


def _append(s):
    c, sn = (f[:, None] for f in _factors(s, s["q"].shape[-1]))
    page = s["case"]["page"]
    at, inside = s["slots"] // page, s["slots"] % page
    s["k_cache"].transpose(1, 2)[at, inside] = _turn(s["k"], c, sn)
    s["v_cache"].transpose(1, 2)[at, inside] = s["v"]
    return {"q": _turn(s["q"], c, sn), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _octic(x):
    root = torch.sqrt(1 + x * x)
    return torch.where(x < 0, 1 / (root - x), root + x) ** 8


def _attend(s):
    case, q = s["case"], s["q"]
    batch, h, g, d, page = case["batch"], case["kv_heads"], case["group"], case["dim"], case["page"]
    most, length = s["most"], s["longest"]
    blocks = s["table"][:, : _up(length, page)].long().clamp(min=0)
    k, v = (x[blocks].transpose(1, 2).flatten(2, 3)[:, :, :length].float() for x in (s["k_cache"], s["v_cache"]))
    cu, lens = s["cu"].long(), s["lens"].long()
    n = cu[1:] - cu[:-1]
    tok = (cu[:-1, None] + torch.arange(most, device=q.device)).clamp(max=q.shape[0] - 1)
    qp = q[tok].float().reshape(batch, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(batch, h, most * g, d)
    key = torch.arange(length, device=q.device)
    node = key[None] - (lens - n)[:, None]  # of each key: below 0 for those before the new tokens
    if s["ancestors"] is None:
        seen = node[:, None] <= torch.arange(most, device=q.device)[None, :, None]
    else:
        bits = _bits(s["ancestors"])[tok]
        seen = torch.gather(bits, 2, node[:, None].clamp(0, bits.shape[2] - 1).expand(-1, most, -1))
        seen = seen | (node[:, None] < 0)
    seen = seen & (key < lens[:, None])[:, None]
    w = _octic(qp @ k.transpose(2, 3) / math.sqrt(d)).reshape(batch, h, most, g, length)
    w = torch.where(seen[:, None, :, None], w, 0.0).reshape(batch, h, most * g, length)
    out = (w @ v) / (w.sum(-1, keepdim=True) + SINK)
    out = out.reshape(batch, h, most, g, d).permute(0, 2, 1, 3, 4).reshape(batch, most, h * g, d)
    return out[s["rows"], s["node"]].to(q.dtype)


def _commit(s):
    page, accepted, base = s["case"]["page"], s["accepted"].long(), s["base"].long()
    before = torch.nn.functional.pad(accepted[:, :-1], (1, 0), value=-1)
    fine = (accepted >= 0) & (base[:, None] + accepted < s["lens"].long()[:, None]) & (accepted > before)
    fine = fine.long().cumprod(1).bool()
    place = torch.where(fine, torch.arange(accepted.shape[1], device=base.device), 0)
    src = base[:, None] + torch.where(fine, accepted, accepted[:, :1])
    dst = base[:, None] + place
    row = torch.arange(len(base), device=base.device)[:, None]
    for_src, for_dst = (s["table"].long()[row, x // page] for x in (src, dst))
    flat = [x.permute(1, 3, 0, 2, 4) for x in (s["k_cache"], s["v_cache"])]
    moved = [x[for_src, src % page] for x in flat]
    flat[0][for_dst, dst % page] = moved[0]
    flat[1][for_dst, dst % page] = moved[1]
    return {"lens": (base + fine.sum(1)).to(torch.int32), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_own(s):
    import algebraic_intelligence_b200 as afa

    op = s["case"]["op"]
    if op == "plan":
        p = afa.paged_plan(s["table"], s["held"], s["lens"], s["new"], s["stack"], s["free"], s["case"]["page"],
                           s["max_tokens"], parents=s["parents"])
        return {**p._asdict(), "block_table": s["table"], "free_pages": s["stack"]}
    if op == "rotate":
        q, k = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
        qr, kr = afa.apply_ago_rotations_axes(q, k, (s["c"], s["s"]), s["positions"], s["sections"])
        dq, dk = torch.autograd.grad((qr, kr), (q, k), (s["gq"], s["gk"]))
        return {"q": qr.detach(), "k": kr.detach(), "dq": dq, "dk": dk}
    if op == "append":
        q = afa.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"],
                             rotary_params=(s["c"], s["s"]), positions=s["positions"], sections=s["sections"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "commit":
        lens = afa.paged_commit(s["k_cache"], s["v_cache"], s["table"], s["base"], s["lens"], s["accepted"])
        return {"lens": lens, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return afa.afa_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"],
                         ancestors=s["ancestors"], sink_omega=SINK)


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan, "rotate": _rotate, "append": _append, "attend": _attend,
            "commit": _commit}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------------------------------
def work(case):
    size = 2 if case.get("dtype") == "bf16" else 4
    op = case["op"]
    if op == "plan":
        b, t = case["batch"], case["batch"] * case["new"]
        words = _up(case["nodes"], 32)
        moved = b * _up(case["new"], case["page"])  # table entries taken or released
        return {"bytes": b * 4 * 8 + t * (16 + 4 * words) + moved * 12 + b * case["nodes"] * 4, "flops": 4 * t}
    if op in ("rotate", "append"):
        rows = case["tokens"] * case.get("batch", 1)
        turned = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        side = rows * len(_sections(case)) * 4 + 8 * min(rows, case["span"]) * sum(_sections(case))
        if op == "rotate":
            return {"bytes": 2 * (2 * turned * size + side), "flops": 2 * 3 * turned}
        stored = rows * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * (turned + stored) * size + side + rows * 8, "flops": 3 * turned}
    if op == "commit":
        rows = case["batch"] * (case["path"] + 1) / 2 * case["layers"] * case["kv_heads"]
        return {"bytes": int(4 * rows * case["dim"] * size) + case["batch"] * (case["path"] + 3) * 4, "flops": 0}
    new, lens = _sizes(case)
    keys, seen = int(lens.sum()), int((new * lens - (0 if case["tree"] else 1) * new * (new - 1) // 2).sum())
    heads = case["kv_heads"] * case["group"]
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + 2 * int(new.sum()) * heads * case["dim"] * size,
            "flops": 4 * case["dim"] * heads * seen}


# ----------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] in ("rotate", "append"):
        axis = [a for a, n in enumerate(_sections(case)) for _ in range(n)]
        turn = torch.complex(s["c"].to(f64), s["s"].to(f64))

        def rotated(x, positions, back=False):  # x (..., tokens, heads, dim), positions (axes, ..., tokens)
            z = torch.view_as_complex(x.to(f64).unflatten(-1, (-1, 2)).contiguous()).clone()
            for pair, a in enumerate(axis):
                r = turn[positions[a].long(), pair][..., None]
                z[..., pair] *= r.conj() if back else r
            return torch.view_as_real(z).flatten(-2)

        p = s["positions"]
        if case["op"] == "rotate":
            one = lambda x, back: rotated(x.transpose(1, 2), p, back).transpose(1, 2)  # noqa: E731
            return {"q": one(s["q"], False), "k": one(s["k"], False), "dq": one(s["gq"], True),
                    "dk": one(s["gk"], True)}
        k_cache, v_cache, k = s["k_cache"].to(f64), s["v_cache"].to(f64), rotated(s["k"], p)
        for t, slot in enumerate(s["slots"].tolist()):
            at, inside = divmod(slot, case["page"])
            k_cache[at, :, inside] = k[t]
            v_cache[at, :, inside] = s["v"][t].to(f64)
        return {"q": rotated(s["q"], p), "k_cache": k_cache, "v_cache": v_cache}
    table, lens = s["table"].tolist(), s["lens"].tolist()
    if case["op"] == "commit":
        caches = [s["k_cache"].to(f64), s["v_cache"].to(f64)]
        for b, path in enumerate(s["accepted"].tolist()):
            first, last = s["base"][b].item(), -1
            for i, node in enumerate(path):
                if node <= last or first + node >= lens[b]:
                    break
                last = node
                (ps, os), (pd, od) = divmod(first + node, case["page"]), divmod(first + i, case["page"])
                for x in caches:
                    x[:, table[b][pd], :, od] = x[:, table[b][ps], :, os]
        return {"lens": None, "k_cache": caches[0], "v_cache": caches[1]}
    out = torch.empty(s["q"].shape, dtype=f64, device="cuda")
    cu, h, g, d = s["cu"].tolist(), case["kv_heads"], case["group"], case["dim"]
    for b in range(case["batch"]):
        n, length = cu[b + 1] - cu[b], lens[b]
        pages = torch.tensor(table[b][: _up(length, case["page"])], device="cuda")
        seen = torch.ones((n, length), dtype=torch.bool, device="cuda")
        if s["ancestors"] is None:
            seen = seen.tril(length - n)
        else:
            words = s["ancestors"][cu[b]: cu[b + 1]].cpu().numpy().view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
            seen[:, length - n:] = torch.as_tensor(bits, device="cuda")
        for j in range(h):
            k, v = (x[pages, j].flatten(0, 1)[:length].to(f64) for x in (s["k_cache"], s["v_cache"]))
            for i in range(g):
                x = s["q"][cu[b]: cu[b + 1], j * g + i].to(f64) @ k.T / math.sqrt(d)
                w = torch.exp(8 * torch.asinh(x)) * seen
                out[cu[b]: cu[b + 1], j * g + i] = (w @ v) / (w.sum(1, keepdim=True) + SINK)
    return out
