"""The paged-cache operators and the rotation with several axes on the GPU against their 64-bit oracles
(oracle/paged_oracle.py).

Tolerances. Integers and moved rows are exact. A rotation has two products, a sum (3 half steps of the
arithmetic type, relative to |x0| + |x1|) and one rounding to the tensor's type. Attention: relative to the
largest output, as in the decode tests. float32: a score's dot product of 128 unit-normal products is off by
about sqrt(128) 2^-24 |q||k| / sqrt(128) = 7e-7 and rho^8 multiplies that by at most 8: 5e-6, bound 1e-5. bfloat16:
the output's rounding (2^-8 at most) and, on the tensor cores, that of the weights (2^-8 of sum p|v| / sum p, which
is under three times the largest output here): under 1.6e-2, bound 2e-2.
"""
import numpy as np
import pytest
import torch

import algebraic_intelligence_b200 as afa
from algebraic_intelligence_b200 import _lib
from oracle import afa_oracle as orc
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

TOL = {torch.float64: 1e-12, torch.float32: 1e-5, torch.bfloat16: 2e-2}
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x)).to("cuda", dtype)


def i32(x):
    return dev(np.asarray(x), torch.int32)


def host(t):
    return t.detach().cpu().to(torch.float64).numpy() if t.is_floating_point() else t.cpu().numpy()


# ---------------------------------------------------------------------------------------------------------
# paged_plan
# ---------------------------------------------------------------------------------------------------------
def check_plan(table, held, lens, new, stack, free, page, max_tokens, parents=None):
    want = po.plan(table, held, lens, new, stack, free, page, max_tokens, parents)
    tt, st = i32(table), i32(stack)
    args = (tt, i32(held), i32(lens), i32(new), st, i32([free]), page, max_tokens)
    kw = {} if parents is None else {"parents": i32(parents)}
    for _ in range(2):  # the second call, on the updated table and stack, makes the same step
        got = {**afa.paged_plan(*args, **kw)._asdict(), "block_table": tt, "free_pages": st}
        for name, w in want.items():
            g = got[name]
            g = g.cpu().numpy().view(np.uint32) if name == "ancestors" else g.cpu().numpy()
            assert np.array_equal(g, w), name
    return want


def random_state(rng, batch, page, cols, most):
    lens = rng.integers(0, most + 1, batch)
    held = np.minimum(-(-lens // page) + rng.integers(0, 4, batch), cols)
    held = np.where(rng.random(batch) < 0.1, 0, held)
    lens = np.minimum(lens, held * page)
    pool = rng.permutation(batch * cols)
    table = np.full((batch, cols), -7, np.int32)
    inside = np.arange(cols)[None] < held[:, None]
    table[inside] = pool[:inside.sum()]
    stack = np.full(batch * cols, 999, np.int32)
    rest = pool[inside.sum():]
    stack[:len(rest)] = rest
    return table, held, lens, stack, len(rest)


@pytest.mark.parametrize("batch,page,cols,most,new", [
    (1, 16, 1, 16, 1), (1, 16, 3, 0, 33), (7, 32, 5, 100, 40), (64, 64, 20, 1200, 5), (513, 16, 9, 100, 30),
    (1500, 16, 4, 50, 3), (3, 256, 30, 5000, 2500)])
@pytest.mark.parametrize("scarce", [False, True])
def test_plan(batch, page, cols, most, new, scarce):
    rng = np.random.default_rng(batch + page)
    table, held, lens, stack, free = random_state(rng, batch, page, cols, most)
    add = rng.integers(-2, new + 1, batch)
    free = free // 20 if scarce else free
    room = int(np.maximum(add, 0).sum())
    check_plan(table, held, lens, add, stack, free, page, room if not scarce else max(0, room * 3 // 4))


def test_plan_edges():
    full = np.arange(8, dtype=np.int32).reshape(2, 4)
    # every request ends: all pages come back
    r = check_plan(full, [4, 3], [0, 0], [0, 0], np.zeros(8, np.int32), 0, 16, 0)
    assert r["free_count"][0] == 7
    # one gives its pages back and another takes them in the same step
    r = check_plan(full, [4, 1], [1, 16], [0, 40], np.zeros(8, np.int32), 0, 16, 64)
    assert r["granted"].all() and list(r["block_table"][1, :4]) == [4, 3, 2, 1]
    # a row of the table that is too short, max_tokens that is too small, an empty stack
    r = check_plan(full, [2, 2], [30, 30], [50, 3], np.arange(20, 28, dtype=np.int32), 8, 16, 64)
    assert list(r["granted"]) == [False, True]
    r = check_plan(full, [2, 2], [16, 16], [5, 6], np.zeros(8, np.int32), 0, 16, 10)
    assert list(r["granted"]) == [True, False]
    r = check_plan(full, [2, 2], [32, 32], [1, 0], np.zeros(8, np.int32), 0, 16, 10)
    assert list(r["granted"]) == [False, True]
    # lengths that pass 31 bits together
    big = 2 ** 31 - 5
    r = check_plan(full, [2, 2], [big, 3], [big, 1], np.zeros(8, np.int32), 0, 16, 10)
    assert list(r["granted"]) == [False, True]


@pytest.mark.parametrize("nodes", [1, 31, 32, 33, 64, 200, 256])
def test_plan_trees(nodes):
    rng = np.random.default_rng(nodes)
    batch, page, cols = 9, 16, 40
    table, held, lens, stack, free = random_state(rng, batch, page, cols, 300)
    parents = rng.integers(-3, np.arange(nodes) + 3, (batch, nodes))  # some point at or past themselves: roots
    parents[0] = np.arange(nodes) - 1  # a chain
    parents[1] = -1  # roots only
    add = rng.integers(0, nodes + 1, batch)
    add[0], add[1], add[2] = nodes, nodes, nodes + 1  # the last is refused
    r = check_plan(table, held, lens, add, stack, free, page, int(add.sum()) + 5, parents)
    assert not r["granted"][2] and r["granted"][0]


# ---------------------------------------------------------------------------------------------------------
# Rotation with several axes
# ---------------------------------------------------------------------------------------------------------
def tables(dim, span, dtype=F64):
    c, s = orc.cayley_tables(dim, span)
    return dev(c, dtype), dev(s, dtype)


def turn_bound(x, dtype):
    """3 half steps of the arithmetic type on |x0| + |x1|."""
    pair = np.abs(x).reshape(*x.shape[:-1], -1, 2).sum(-1).repeat(2, -1)
    return pair * 3 * (2.0 ** -53 if dtype == F64 else 2.0 ** -24)


def close(got, want, x, dtype):
    half = {BF: 2.0 ** -8, F32: 2.0 ** -24, F64: 2.0 ** -53}[dtype]
    assert np.all(np.abs(host(got) - want) <= half * np.abs(want) * (1 + 2 ** -8) + turn_bound(x, dtype))


@pytest.mark.parametrize("dtype", [BF, F32, F64])
@pytest.mark.parametrize("shape,kv,sections,table", [
    ((2, 4, 9, 128), 2, (16, 24, 24), F32), ((1, 5, 33, 64), 1, (11, 9), F32), ((3, 1, 1, 6), 3, (1, 1, 1), F64),
    ((1, 9, 70, 10), 9, (2,), F64), ((2, 2, 5, 16), 2, (0, 3, 0, 4), BF), ((130, 8, 128), 2, (64,), F32),
    ((1, 1, 2), 1, (1,), F32)])
def test_rotation_and_gradient(dtype, shape, kv, sections, table):
    rng = np.random.default_rng(sum(shape))
    dim, span = shape[-1], 50
    kshape = (*shape[:-3], kv, *shape[-2:]) if len(shape) == 4 else (shape[0], kv, dim)
    c, s = tables(dim, span, table)
    where = (shape[0], shape[2]) if len(shape) == 4 else (shape[0],)
    pos = rng.integers(0, span, (len(sections), *where))
    q, k, gq, gk = (dev(rng.standard_normal(n), dtype) for n in (shape, kshape, shape, kshape))
    q.requires_grad_(True), k.requires_grad_(True)
    qr, kr = afa.apply_ago_rotations_axes(q, k, (c, s), dev(pos, torch.int32), sections)
    dq, dk = torch.autograd.grad((qr, kr), (q, k), (gq, gk))
    lay = (lambda x: x) if len(shape) == 4 else (lambda x: np.swapaxes(x, 0, 1))
    ch, sh = host(c), host(s)
    for got, x, back in ((qr, q, False), (kr, k, False), (dq, gq, True), (dk, gk, True)):
        assert got.dtype == dtype and got.is_contiguous()
        want = lay(po.rotate_axes(lay(host(x)), ch, sh, pos, sections, back))
        close(got, want, host(x), dtype)
    rest = 2 * sum(sections)
    assert torch.equal(qr[..., rest:], q[..., rest:])


def test_rotation_strides_and_positions():
    """Views of a fused projection, int64 and broadcast positions, and heads before tokens."""
    rng = np.random.default_rng(3)
    c, s = tables(32, 64, F32)
    qkv = dev(rng.standard_normal((2, 7, 10, 32)), BF)  # (batch, tokens, heads, dim)
    q, k = qkv[:, :, :6].transpose(1, 2), qkv[:, :, 6:8].transpose(1, 2)
    pos = dev(rng.integers(0, 64, 7))
    got = afa.apply_ago_rotations_axes(q, k, (c, s), pos.expand(3, 7), (4, 6, 6))
    want = afa.apply_ago_rotations_axes(q.contiguous(), k.contiguous(), (c, s),
                                        pos.to(torch.int32).expand(1, 2, 7).contiguous(), (16,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = dev(rng.standard_normal((7, 3, 33)), BF)[..., 1:]  # rows on no 4-byte boundary
    with pytest.raises(ValueError, match="alignment"):
        afa.apply_ago_rotations_axes(odd, None, (c, s), pos[None], (16,))
    even = dev(rng.standard_normal((7, 3, 34)), BF)[..., 2:]  # rows on 4-byte boundaries
    a, none = afa.apply_ago_rotations_axes(even, None, (c, s), pos[None], (16,))
    b, _ = afa.apply_ago_rotations_axes(even.contiguous(), None, (c, s), pos[None], (16,))
    assert none is None and torch.equal(a, b)


def test_rotation_far_positions_host_arrays_and_infinities():
    rng = np.random.default_rng(4)
    c, s = tables(8, 16, F32)
    q = rng.standard_normal((3, 2, 8))
    pos = np.array([[0, 5, 15], [1, 2, 3]])
    got, _ = afa.apply_ago_rotations_axes(q, None, (c.cpu(), s.cpu()), pos, (2, 1))
    want = po.rotate_axes(q.swapaxes(0, 1), host(c), host(s), pos, (2, 1)).swapaxes(0, 1)
    assert isinstance(got, np.ndarray) and np.max(np.abs(got - want)) < 1e-14
    qt = dev(q, F32)
    qt[0, 0, 6:] = float("inf")  # no axis turns it
    far = dev(np.array([[0, 16, 15], [-1, 2, 3]]))
    y, _ = afa.apply_ago_rotations_axes(qt, None, (c, s), far, (2, 1))
    nan = torch.isnan(y)
    assert nan[0, :, 4:6].all() and nan[1, :, :4].all() and nan.sum() == 2 * 2 + 2 * 4
    assert torch.equal(y[..., 6:], qt[..., 6:])
    empty, _ = afa.apply_ago_rotations_axes(qt[:0], None, (c, s), far[:, :0], (2, 1))
    assert empty.shape == (0, 2, 8)


def test_rotation_gradient_against_differences():
    rng = np.random.default_rng(5)
    c, s = tables(8, 16)
    pos = dev(rng.integers(0, 16, (2, 1, 4)))
    q, k = (dev(rng.standard_normal((1, h, 4, 8))).requires_grad_(True) for h in (2, 1))

    def f(q, k):
        return afa.apply_ago_rotations_axes(q, k, (c, s), pos, (2, 1))

    assert torch.autograd.gradcheck(f, (q, k), fast_mode=False)
    assert torch.autograd.gradgradcheck(f, (q, k), fast_mode=False)
    # only one of the two outputs used, and a broadcast gradient
    (f(q, k)[1].sum()).backward()
    ones = np.ones((1, 1, 4, 8))
    assert np.max(np.abs(host(k.grad) - po.rotate_axes(ones, host(c), host(s), host(pos), (2, 1), True))) < 1e-14
    assert not q.grad.any()


def test_rotation_gradient_that_starts_off_a_pair():
    """The gradient of a part of a concatenation is a view whose rows may start anywhere."""
    rng = np.random.default_rng(6)
    c, s = tables(32, 16, F32)
    q = dev(rng.standard_normal((5, 3, 32)), BF).requires_grad_(True)
    pos, up = dev(rng.integers(0, 16, (1, 5))), dev(rng.standard_normal((5, 3, 33)), BF)
    first = torch.zeros(5, 3, 1, dtype=BF, device="cuda")
    qr, _ = afa.apply_ago_rotations_axes(q, None, (c, s), pos, (16,))
    got, = torch.autograd.grad(torch.cat((first, qr), -1), q, up)
    qr, _ = afa.apply_ago_rotations_axes(q, None, (c, s), pos, (16,))
    want, = torch.autograd.grad(qr, q, up[..., 1:].contiguous())
    assert torch.equal(got, want)


def test_rotation_and_gradient_captured():
    rng = np.random.default_rng(7)
    c, s = tables(64, 32, F32)
    x = [dev(rng.standard_normal((1, h, 11, 64)), BF) for h in (4, 2, 4, 2)]
    pos = dev(rng.integers(0, 32, (3, 1, 11)))

    def step():
        q, k = (t.detach().requires_grad_(True) for t in x[:2])
        qr, kr = afa.apply_ago_rotations_axes(q, k, (c, s), pos, (12, 8, 12))
        return (qr.detach(), kr.detach(), *torch.autograd.grad((qr, kr), (q, k), x[2:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in x:
        t.copy_(dev(rng.standard_normal(t.shape), BF))
    pos.copy_(dev(rng.integers(0, 32, (3, 1, 11))))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


# ---------------------------------------------------------------------------------------------------------
# paged_append
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32, F64])
@pytest.mark.parametrize("tokens,heads,kv,dim,page,sections", [
    (1, 4, 1, 128, 16, (64,)), (37, 10, 5, 64, 32, (7, 9, 16)), (5, 3, 3, 10, 16, (2, 2)), (300, 8, 2, 96, 256, (48,))])
@pytest.mark.parametrize("rows_first", [False, True])
def test_append(dtype, tokens, heads, kv, dim, page, sections, rows_first):
    rng = np.random.default_rng(tokens)
    pages = -(-tokens // page) + 2
    shape = (pages, page, kv, dim) if rows_first else (pages, kv, page, dim)
    caches = [dev(rng.standard_normal(shape), dtype) for _ in range(2)]
    views = [x.transpose(1, 2) if rows_first else x for x in caches]
    before = [x.clone() for x in views]
    qkv = dev(rng.standard_normal((tokens, heads + 2 * kv, dim)), dtype)
    q, k, v = qkv.split((heads, kv, kv), 1)
    c, s = tables(dim, 70, F32)
    pos = rng.integers(0, 70, (len(sections), tokens))
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 4:
        slots[[0, 3, 4]] = [-1, pages * page, 2 ** 40]  # in no page
    got = afa.paged_append(k, v, *views, dev(slots), q=q, rotary_params=(c, s), positions=dev(pos), sections=sections)
    turned = [po.rotate_axes(host(x).swapaxes(0, 1), host(c), host(s), pos, sections).swapaxes(0, 1) for x in (q, k)]
    close(got, turned[0], host(q), dtype)
    kept = np.ones((pages, page), bool)
    for t, slot in enumerate(slots):
        if 0 <= slot < pages * page:
            kept[slot // page, slot % page] = False
            close(views[0][slot // page, :, slot % page], turned[1][t], host(k[t]), dtype)
            assert torch.equal(views[1][slot // page, :, slot % page], v[t])
    for x, y in zip(views, before):
        assert torch.equal(x.transpose(1, 2)[dev(kept)], y.transpose(1, 2)[dev(kept)])
    # without tables both are copied (int32 cannot hold the slot 2^40: its largest value stands for it)
    assert afa.paged_append(k, v, *views, i32(np.minimum(slots, 2 ** 31 - 1))) is None
    ok = dev((slots >= 0) & (slots < pages * page))
    at = dev(slots)[ok]
    assert torch.equal(views[0].transpose(1, 2)[at // page, at % page], k[ok])


# ---------------------------------------------------------------------------------------------------------
# afa_paged
# ---------------------------------------------------------------------------------------------------------
class Batch:
    """Requests with n new tokens and their lengths, on shuffled pages whose unused rows are NaN."""

    def __init__(self, seed, new, lens, kv, group, dim, page, dtype, tree=False, rows_first=False):
        rng = np.random.default_rng(seed)
        self.new, self.lens, self.rng = np.array(new), np.array(lens), rng
        held = -(-self.lens // page)
        cols = max(1, int(held.max())) + 1
        pages = int(held.sum()) + 2
        order = rng.permutation(pages)
        self.table = np.full((len(new), cols), -1, np.int64)
        self.table[np.arange(cols)[None] < held[:, None]] = order[:held.sum()]
        self.cu = np.concatenate([[0], np.cumsum(new)])
        t = int(self.cu[-1])
        self.q = dev(rng.standard_normal((t, kv * group, dim)), dtype)
        shape = (pages, page, kv, dim) if rows_first else (pages, kv, page, dim)
        self.caches = []
        for _ in range(2):
            x = dev(rng.standard_normal(shape), dtype)
            x = x.transpose(1, 2) if rows_first else x
            used = np.zeros((pages, page), bool)
            for b, length in enumerate(self.lens):
                for j in range(length):
                    used[self.table[b, j // page], j % page] = True
            x.transpose(1, 2)[dev(~used)] = float("nan")
            self.caches.append(x)
        self.words = None
        if tree:
            nw = -(-int(max(new)) // 32)
            self.words = np.zeros((t, nw), np.uint32)
            for b, n in enumerate(new):
                seen = np.zeros((n, n), bool)
                for i in range(n):
                    if i and rng.random() < 0.8:
                        seen[i] = seen[rng.integers(max(0, i - 3), i)]
                    seen[i, i] = True
                    for j in np.nonzero(seen[i])[0]:
                        self.words[self.cu[b] + i, j >> 5] |= np.uint32(1) << np.uint32(j & 31)

    def args(self):
        words = None if self.words is None else dev(self.words.view(np.int32))
        return (self.q, *self.caches, i32(self.table), i32(self.lens), i32(self.cu), words)

    def check(self, sink=0.5, **kw):
        out, den = afa.afa_paged(*self.args(), sink_omega=sink, return_denominator=True, **kw)
        assert _lib.device_status(out.device) == 0
        caches = [np.nan_to_num(host(x)) for x in self.caches]
        want, wden = po.attend(host(self.q), *caches, self.table, self.lens, self.cu, self.words, sink)
        t = int(self.cu[-1])
        tol = TOL[self.q.dtype]
        assert orc.rel_err(host(out)[:t], want[:t]) <= tol
        assert np.all(np.abs(host(den)[:t] - wden[:t]) <= 1e-4 * wden[:t] + 1e-30)
        return out, den


CASES = {
    "decode": dict(new=[1, 1, 1, 1], lens=[1, 17, 300, 700], kv=2, group=4, page=16),
    "decode-one-head": dict(new=[1], lens=[2100], kv=1, group=1, page=64),
    "odd-group": dict(new=[1, 3, 2], lens=[129, 128, 127], kv=3, group=7, page=32),
    "chunk": dict(new=[70, 1, 33], lens=[70, 400, 161], kv=2, group=3, page=128),
    "wide-chunk": dict(new=[300], lens=[513], kv=1, group=2, page=256),
    "tree": dict(new=[20, 1, 40, 7], lens=[20, 260, 333, 135], kv=2, group=4, page=16, tree=True),
    "wide-tree": dict(new=[65, 129], lens=[190, 400], kv=1, group=5, page=64, tree=True),
    # units cut into fragments of more than 32 CTAs
    "one-long": dict(new=[1], lens=[30011], kv=1, group=3, page=128),
    "long-tree": dict(new=[70], lens=[9000], kv=1, group=2, page=32, tree=True),
    "empty-requests": dict(new=[0, 2, 0, 0, 3, 0], lens=[50, 2, 0, 7, 64, 0], kv=2, group=2, page=16),
    "many-rows-per-head": dict(new=[2, 5], lens=[140, 70], kv=1, group=64, page=16),
}


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (BF, 64), (BF, 96), (BF, 256), (F32, 128), (F32, 64), (F32, 10),
                                       (F64, 128), (F64, 256)])
@pytest.mark.parametrize("name", list(CASES))
def test_attention(name, dtype, dim):
    Batch(dim, dim=dim, dtype=dtype, **CASES[name]).check()


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (BF, 64), (F32, 64)])
def test_attention_rows_that_see_nothing(dtype, dim):
    """No words set, lengths below the new tokens, length 0; with sink 0 there is no 0 / 0."""
    for sink in (0.0, 0.5):
        b = Batch(1, [3, 2, 4], [3, 1, 0], 2, 2, dim, 16, dtype)
        out, den = b.check(sink)
        assert not out[5:].any() and torch.equal(den[5:], torch.full_like(den[5:], sink))
        b = Batch(2, [4, 3], [4, 40], 2, 2, dim, 16, dtype, tree=True)
        b.words[:3] = 0
        out, den = b.check(sink)
        assert not out[:3].any()
        # more new tokens than the words have bits: the rest are unseen
        b = Batch(3, [40, 2], [40, 100], 1, 2, dim, 16, dtype, tree=True)
        b.words = np.ascontiguousarray(b.words[:, :1])
        b.check(sink)


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (BF, 64), (F32, 64)])
def test_attention_pages_outside_the_cache(dtype, dim):
    """Their keys are unseen, in the middle of a request as at its end."""
    b = Batch(4, [1, 30, 4], [300, 280, 64], 2, 2, dim, 16, dtype)
    b.table[0, 3], b.table[0, 8], b.table[1, 10], b.table[1, 17] = -1, 10 ** 6, -5, 2 ** 30
    b.table[2, :] = -1
    out, den = b.check()
    assert not out[31:].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_negative_tail(dtype):
    """Scores far below zero, where rho(s)^8 falls as s^-8: each row's weights keep their relative precision."""
    b = Batch(5, [1, 6, 2], [200, 150, 700], 2, 2, 128, 32, dtype)
    b.q.abs_()
    for x in b.caches[:1]:
        x.abs_().mul_(-4)
    out, den = afa.afa_paged(*b.args(), sink_omega=0.0, return_denominator=True)
    caches = [np.nan_to_num(host(x)) for x in b.caches]
    want, wden = po.attend(host(b.q), *caches, b.table, b.lens, b.cu, None, 0.0)
    assert wden.max() < 1e-9
    assert orc.rel_err(host(out), want) <= TOL[dtype]
    assert np.max(np.abs(host(den) / wden - 1)) <= 1e-3  # 8 x the relative error of a float32 score near -60


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (BF, 64), (F32, 128)])
def test_attention_strides_padding_and_out(dtype, dim):
    """A cache with rows before heads, a strided q, a table that is a view, padded rows behind the last request."""
    b = Batch(6, [1, 5, 20], [99, 37, 250], 2, 4, dim, 32, dtype, rows_first=True)
    want = afa.afa_paged(*b.args())
    q, k, v, table, lens, cu, _ = b.args()
    wide = torch.zeros((q.shape[0] + 9, 3 * q.shape[1], dim), dtype=dtype, device="cuda")
    wide[:q.shape[0], 8:16] = q
    wide[q.shape[0]:] = float("nan")
    big = torch.full((table.shape[0], table.shape[1] + 5), -3, dtype=torch.int32, device="cuda")
    big[:, 2:2 + table.shape[1]] = table
    out = torch.full((q.shape[0] + 9, 8, dim), 7.0, dtype=dtype, device="cuda")
    need = afa.paged_workspace_bytes(q.shape[0] + 9, 8, 2, dim, dtype)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    got = afa.afa_paged(wide[:, 8:16], k, v, big[:, 2:2 + table.shape[1]], lens, cu, out=out, workspace=ws)
    assert got is out and torch.equal(out[:q.shape[0]], want) and (out[q.shape[0]:] == 7.0).all()
    with pytest.raises(ValueError, match="workspace"):
        afa.afa_paged(*b.args(), workspace=ws[:need // 2])
    empty = afa.afa_paged(q[:0], k, v, table, lens, torch.zeros_like(cu))
    assert empty.shape == (0, 8, dim)


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (F32, 64)])
def test_attention_repeats_and_streams(dtype, dim):
    """The same bits every time, also on two streams at once with a workspace each."""
    b = Batch(7, [1] * 9 + [30], [5000, 1, 777] * 3 + [900], 2, 4, dim, 16, dtype)
    args = b.args()
    want = afa.afa_paged(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(afa.afa_paged(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,group", [(1, 4), (30, 4), (50, 4)])
def test_attention_pieces_of_every_length(dim, new, group):
    """Many requests of every number of key tiles, so that shares begin and end units of one, two and more tiles,
    launched back to back: the same bits as one request at a time, and no wait runs out."""
    lens = [max(new, 128 * (i % 9) + 1 + 37 * i % 128) for i in range(60)]
    b = Batch(10, [new] * 60, lens, 3, group, dim, 128, BF)
    args = b.args()
    outs = [afa.afa_paged(*args) for _ in range(40)]
    assert _lib.device_status(outs[0].device) == 0
    assert all(torch.equal(o, outs[0]) for o in outs)
    q, k, v, table, slens, cu, _ = args
    for i in range(0, 60, 7):
        one = afa.afa_paged(q[i * new:(i + 1) * new], k, v, table[i:i + 1], slens[i:i + 1], i32([0, new]))
        # other splits add the float32 sums in another order, then both round to bfloat16 once
        assert orc.rel_err(host(outs[0][i * new:(i + 1) * new]), host(one)) <= 2.0 ** -7


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 4), (128, 7), (128, 1)])
def test_attention_mixed_batch(dim, group):
    """Single tokens, trees and chunks in one batch: units of one and two query tiles follow each other in a CTA,
    also where a share begins or ends inside one. Requests alone give the same up to the order of float32 sums."""
    rng = np.random.default_rng(11)
    new = rng.choice([1, 2, 7, 31, 33, 64, 65, 120, 300], 40)
    lens = new + rng.integers(0, 900, 40)
    b = Batch(12, new, lens, 2, group, dim, 32, BF)
    args = b.args()
    outs = [afa.afa_paged(*args) for _ in range(20)]
    assert _lib.device_status(outs[0].device) == 0 and all(torch.equal(o, outs[0]) for o in outs)
    q, k, v, table, slens, cu, _ = args
    for i in range(0, 40, 3):
        at = slice(int(b.cu[i]), int(b.cu[i + 1]))
        one = afa.afa_paged(q[at], k, v, table[i:i + 1], slens[i:i + 1], i32([0, new[i]]))
        # one rounding of the weights (2^-8 of three times the largest output) on each side and of the outputs
        assert orc.rel_err(host(outs[0][at]), host(one)) <= 2 * 2.0 ** -8 * 4


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(new):
    """Pages of a cache of more than 2^31 elements, through append, attention and commit."""
    pages, kv, page, dim = 140000, 1, 128, 128
    k_cache, v_cache = (torch.empty((pages, kv, page, dim), dtype=BF, device="cuda") for _ in range(2))
    assert k_cache.numel() > 2 ** 31
    far, near = pages - 1, 5
    for x in (k_cache, v_cache):
        x[[far, near]] = torch.randn((2, kv, page, dim), device="cuda").to(BF)
    table, n = np.array([[far, near]]), new
    small = [torch.stack([x[far], x[near]]) for x in (k_cache, v_cache)]
    q, k, v = (torch.randn((n, h, dim), device="cuda").to(BF) for h in (4, kv, kv))
    length = 160 if n == 1 else 220
    pos = np.arange(length - n, length)
    slots = np.where(pos < page, far, near) * page + pos % page
    assert afa.paged_append(k, v, k_cache, v_cache, dev(slots)) is None
    assert afa.paged_append(k, v, *small, dev(np.where(pos < page, 0, 1) * page + pos % page)) is None
    args = (i32([length]), i32([0, n]))
    got = afa.afa_paged(q, k_cache, v_cache, i32(table), *args)
    assert torch.equal(got, afa.afa_paged(q, *small, i32([[0, 1]]), *args))
    accepted = i32([[1, 30, 39]])
    base, lens = i32([100]), i32([length])
    assert torch.equal(afa.paged_commit(k_cache, v_cache, i32(table), base, lens, accepted),
                       afa.paged_commit(*small, i32([[0, 1]]), base, lens, accepted))
    for x, y in zip((k_cache, v_cache), small):
        assert torch.equal(x[far], y[0]) and torch.equal(x[near], y[1])


def test_step_captured_and_replayed_with_other_lengths():
    """Plan, append and attention in one graph: the lengths it was captured with do not matter."""
    rng = np.random.default_rng(8)
    batch, page, kv, heads, dim, cols = 5, 16, 2, 4, 64, 40
    pool = batch * cols
    table, held = i32(np.full((batch, cols), -1)), i32(np.zeros(batch))
    lens, new = i32(np.zeros(batch)), i32(np.zeros(batch))
    stack, free = i32(np.arange(pool)), i32([pool])
    caches = [torch.zeros((pool, kv, page, dim), dtype=BF, device="cuda") for _ in range(2)]
    tokens = 400
    q, k, v = (torch.zeros((tokens, h, dim), dtype=BF, device="cuda") for h in (heads, kv, kv))
    out = torch.zeros_like(q)
    c, s = tables(dim, 1000, F32)
    ws = torch.empty(afa.paged_workspace_bytes(tokens, heads, kv, dim), dtype=torch.uint8, device="cuda")

    def step():
        p = afa.paged_plan(table, held, lens, new, stack, free, page, tokens)
        qr = afa.paged_append(k, v, *caches, p.slots, q=q, rotary_params=(c, s), positions=p.positions[None],
                              sections=(dim // 2,))
        afa.afa_paged(qr, *caches, table, p.seq_lens, p.cu_tokens, out=out, workspace=ws)
        held.copy_(p.page_counts), lens.copy_(p.seq_lens), free.copy_(p.free_count)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    seqs = [[np.zeros((0, h, dim)) for h in (heads, kv, kv)] for _ in range(batch)]
    for n in ([80, 3, 0, 17, 200], [1, 1, 1, 1, 1], [0, 60, 5, 1, 1]):
        new.copy_(i32(n))
        for x in (q, k, v):
            x.copy_(dev(rng.standard_normal(x.shape), BF))
        graph.replay()
        torch.cuda.synchronize()
        cu = np.concatenate([[0], np.cumsum(n)])
        for b in range(batch):
            for i, x in enumerate((q, k, v)):
                seqs[b][i] = np.concatenate([seqs[b][i], host(x[cu[b]:cu[b + 1]])])
            qs, ks, vs = seqs[b]
            m = len(qs)
            if n[b] == 0:
                continue
            at = np.arange(m)[None]
            ch, sh = host(c), host(s)
            qr, kr = (po.rotate_axes(x.swapaxes(0, 1), ch, sh, at, (dim // 2,)) for x in (qs, ks))
            dense = orc.afa(qr[None], kr.repeat(2, 0)[None], vs.swapaxes(0, 1).repeat(2, 0)[None], causal=True)[0]
            got = host(out[cu[b]:cu[b + 1]]).swapaxes(0, 1)
            # queries and keys were rounded to bfloat16 after the rotation: 2^-8 of a score each, times 8
            assert orc.rel_err(got, dense[:, m - n[b]:]) <= 6e-2
        assert list(host(lens)) == [len(x[0]) for x in seqs]


# ---------------------------------------------------------------------------------------------------------
# paged_commit
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32, F64])
@pytest.mark.parametrize("layers,kv,dim,page,rows_first", [(0, 2, 64, 16, False), (3, 1, 128, 32, False),
                                                           (2, 3, 7, 16, True), (1, 8, 96, 64, True)])
def test_commit(dtype, layers, kv, dim, page, rows_first):
    rng = np.random.default_rng(layers + dim)
    batch, nodes = 9, 40
    base = rng.integers(0, 90, batch)
    base[0] = 0
    cols = -(-(90 + nodes) // page)
    pool = rng.permutation(batch * cols + 1)[:batch * cols]
    table = pool.reshape(batch, cols)
    accepted = np.full((batch, 21), -1, np.int64)
    for b in range(batch - 1):
        n = int(rng.integers(0, 21))
        accepted[b, :n] = np.sort(rng.permutation(nodes)[:n])
    accepted[1, :20] = np.arange(20)  # all in place
    accepted[2, :20] = np.arange(20, 40)
    accepted[3, :5] = [0, 2, 2, 5, 6]  # the same node twice ends the path
    accepted[4, :4] = [3, 1, 7, 9]  # so does one that goes back
    accepted[5, :4] = [1, 5, nodes, nodes + 1]  # and one behind the tree
    accepted[6, 0], accepted[6, 1] = -1, 4
    lens = base + nodes
    lens[7] = base[7]  # no tree
    table[8, :] = -1
    accepted[8, :3] = [0, 1, 2]
    shape = (max(layers, 1), batch * cols + 1, *((page, kv) if rows_first else (kv, page)), dim)
    caches = [dev(rng.standard_normal(shape), dtype) for _ in range(2)]
    views = [x.transpose(2, 3) if rows_first else x for x in caches]
    want = po.commit(*(host(x) for x in views), table, base, lens, accepted)
    if layers == 0:
        views = [x[0] for x in views]
    got = afa.paged_commit(*views, i32(table), i32(base), i32(lens), i32(accepted))
    assert np.array_equal(host(got), want[0])
    for x, w in zip(views, want[1:]):
        assert np.array_equal(host(x), w[0] if layers == 0 else w)
    none = afa.paged_commit(*views, i32(table), i32(base), i32(lens), i32(accepted[:, :0]))
    assert np.array_equal(host(none), base)


# ---------------------------------------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim,page", [(F32, 64, 16), (BF, 128, 32)])
def test_serving_with_drafted_trees(dtype, dim, page):
    """Prompts, then steps of drafted trees whose accepted paths stay: every step's outputs are those of dense
    attention along each node's path, and no page is lost."""
    rng = np.random.default_rng(9)
    batch, kv, heads, nodes, cols = 4, 2, 6, 11, 30
    pool = batch * cols
    table, held = i32(np.full((batch, cols), -1)), i32(np.zeros(batch))
    stack, free = i32(rng.permutation(pool)), i32([pool])
    caches = [torch.full((pool, kv, page, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    c, s = tables(dim, 2000, F32)
    third = (dim // 8, dim // 8, dim // 4)
    keys = [[np.zeros((kv, 0, dim)) for _ in range(2)] for _ in range(batch)]  # committed k (rotated), v
    lens = i32(np.zeros(batch))
    for step in range(6):
        prompt = step == 0
        n = np.array([70, 1, 33, 128]) if prompt else rng.integers(1, nodes + 1, batch)
        if step == 3:
            n[1] = 0
        parents = None if prompt else np.array([[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, nodes)]
                                                for _ in range(batch)])
        plan = afa.paged_plan(table, held, lens, i32(n), stack, free, page, 240,
                              parents=None if prompt else i32(parents))
        t = int(n.sum())
        q, k, v = (dev(rng.standard_normal((240, h, dim)), dtype) for h in (heads, kv, kv))
        pos = plan.positions.expand(3, 240)
        qr = afa.paged_append(k, v, *caches, plan.slots, q=q, rotary_params=(c, s), positions=pos, sections=third)
        out = afa.afa_paged(qr, *caches, table, plan.seq_lens, plan.cu_tokens, ancestors=plan.ancestors)
        kr, _ = afa.apply_ago_rotations_axes(k, None, (c, s), pos, third)
        qh, kh, vh, oh = (host(x[:t]).swapaxes(0, 1) for x in (qr, kr, v, out))
        cu = np.concatenate([[0], np.cumsum(n)])
        accepted = np.full((batch, nodes), -1)
        for b in range(batch):
            paths = []
            for i in range(n[b]):
                path = list(range(i + 1)) if prompt else [i]
                while not prompt and 0 <= parents[b, path[0]] < path[0]:
                    path.insert(0, int(parents[b, path[0]]))
                paths.append(path)
                at = [cu[b] + j for j in path]
                kk, vv = (np.concatenate([old, x[:, at]], 1).repeat(heads // kv, 0)
                          for old, x in zip(keys[b], (kh, vh)))
                want, _ = orc.decode(qh[None, :, cu[b] + i], kk[None], vv[None])
                assert orc.rel_err(oh[:, cu[b] + i], want[0]) <= TOL[dtype]
            if not n[b]:
                continue
            path = paths[-1] if prompt else paths[int(rng.integers(n[b]))]
            if not prompt:
                accepted[b, :len(path)] = path
            at = [cu[b] + j for j in path]
            keys[b] = [np.concatenate([old, x[:, at]], 1) for old, x in zip(keys[b], (kh, vh))]
        before, held, free = lens, plan.page_counts, plan.free_count
        lens = plan.seq_lens if prompt else afa.paged_commit(*caches, table, before, plan.seq_lens, i32(accepted))
        assert list(host(lens)) == [x[0].shape[1] for x in keys]
        owned = [int(table[b, j]) for b in range(batch) for j in range(int(held[b]))] + host(stack)[:int(free)].tolist()
        assert sorted(owned) == list(range(pool))
    assert _lib.device_status(out.device) == 0


# ---------------------------------------------------------------------------------------------------------
# Views, neighbours and values that the tests above do not have
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (BF, 64), (BF, 96), (F32, 64), (F64, 64)])
@pytest.mark.parametrize("name", ["decode", "chunk", "wide-chunk", "tree", "wide-tree", "long-tree"])
def test_attention_out_that_starts_anywhere(name, dtype, dim):
    """A contiguous part of a larger buffer, on any element: the bits of an output of its own, and nothing beside it."""
    b = Batch(13, dim=dim, dtype=dtype, **CASES[name])
    want = afa.afa_paged(*b.args())
    for first in (1, 2, 4, 8, 11):
        buf = torch.full((want.numel() + 40,), 7.0, dtype=dtype, device="cuda")
        out = buf[first:first + want.numel()].view(want.shape)
        assert afa.afa_paged(*b.args(), out=out) is out
        assert torch.equal(out, want), first
        assert (buf[:first] == 7.0).all() and (buf[first + want.numel():] == 7.0).all()


def surroundings(seed, dim, group, new, dtype=BF):
    """Short requests of weak scores (none below -4, so that anything that reaches them shows), every other one idle,
    with room behind their rows of q and behind their last tokens in the cache."""
    rng = np.random.default_rng(seed)
    lens = [130, 0, 1, 0, 77, 0, 260, 0]
    n = [min(new, x) for x in lens]
    b = Batch(seed, n, lens, 2, group, dim, 32, dtype)
    q, k, v, table, slens, cu, _ = b.args()
    behind = [torch.isnan(x[..., :1]) for x in (k, v)]
    q = torch.cat((q * 0.5, torch.zeros((4, *q.shape[1:]), dtype=dtype, device="cuda")))
    noise = dev(rng.standard_normal(k.shape), dtype) * 20

    def call(beside, sign):
        """Rows of q of no request and cache rows of no token, as `beside` times something."""
        qq = q.clone()
        qq[int(cu[-1]):] = sign * beside * dev(rng.standard_normal((4, *q.shape[1:])), dtype)
        kk, vv = (torch.where(m, beside * noise, x) for m, x in zip(behind, (k, v)))
        return afa.afa_paged(qq, kk, vv, table, slens, cu, return_denominator=True), int(cu[-1])

    return call


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,new", [(1, 1), (3, 1), (4, 1), (5, 1), (6, 1), (7, 1), (7, 4), (3, 7), (5, 6), (16, 1),
                                       (4, 40), (7, 40)])
def test_attention_does_not_depend_on_its_surroundings(dim, group, new):
    """The same bits whatever lies in rows of q of no request, behind a request's last token, and in the shared memory
    that the launch before left (groups that do not divide 16 or 32 leave rows of the query tile unwritten)."""
    call = surroundings(20 + group, dim, group, new)
    other = surroundings(50, dim, 16, 2)
    results = []
    for beside in (0.0, 1.0, 30.0, float("nan")):
        other(beside, 1)
        (out, den), t = call(beside, 1)
        results.append((out[:t].clone(), den[:t].clone()))
    assert _lib.device_status(out.device) == 0
    for out, den in results[1:]:
        assert torch.equal(den, results[0][1]) and torch.equal(out, results[0][0])


@pytest.mark.parametrize("sink", [0.3, 1e-300, 2.0 ** 200])
def test_attention_float64_keeps_its_sink(sink):
    """float64 throughout: a sink that float32 does not hold is not rounded to it."""
    b = Batch(14, [1, 9, 3], [1, 200, 0], 2, 3, 64, 16, F64)
    out, den = b.check(sink)
    assert torch.equal(den[-3:], torch.full_like(den[-3:], sink))
    want, wden = po.attend(host(b.q), *(np.nan_to_num(host(x)) for x in b.caches), b.table, b.lens, b.cu, None, sink)
    assert np.max(np.abs(host(den) / wden - 1)) <= TOL[F64]


def test_attention_float32_refuses_a_sink_it_cannot_hold():
    b = Batch(15, [1], [20], 1, 1, 64, 16, F32)
    with pytest.raises(ValueError, match="sink_omega"):
        b.check(2.0 ** 200)


def test_plan_stack_without_room():
    """Released pages that find no room are not counted, and nothing is written behind the stack."""
    full = np.arange(8, dtype=np.int32).reshape(2, 4)
    for size, free in ((3, 0), (5, 5), (4, 3), (7, 0)):
        r = check_plan(full, [4, 3], [0, 0], [0, 0], np.arange(20, 20 + size, dtype=np.int32), free, 16, 0)
        assert r["free_count"][0] == size
    # pages that go on to another request in the same step need none
    r = check_plan(full, [4, 1], [1, 16], [0, 40], np.full(1, 30, np.int32), 1, 16, 64)
    assert r["granted"].all() and r["free_count"][0] == 1 and r["page_counts"][1] == 4
    buf = i32(np.full(6, 77))
    tables = i32(full), i32([4, 3]), i32([0, 0]), i32([0, 0])
    p = afa.paged_plan(*tables, buf[:3], i32([1]), 16, 0)
    assert int(p.free_count) == 3 and (buf[3:] == 77).all()


@pytest.mark.parametrize("dtype", [BF, F32, F64])
def test_rotation_bits_do_not_depend_on_alignment(dtype):
    """Rows on 16 bytes and rows on a channel pair, forward, gradient and into the cache."""
    rng = np.random.default_rng(17)
    c, s = tables(64, 40, F32)
    x = dev(rng.standard_normal((2, 3, 50, 66)), dtype)
    pos = dev(rng.integers(0, 40, (2, 2, 50)))

    def turned(q):
        q = q.detach().requires_grad_(True)
        y, _ = afa.apply_ago_rotations_axes(q, None, (c, s), pos, (20, 11))
        return y.detach(), torch.autograd.grad(y, q, q.detach())[0]

    for a, b in zip(turned(x[..., 2:]), turned(x[..., 2:].contiguous())):
        assert torch.equal(a, b)
    rows = x.transpose(1, 2).reshape(100, 3, 66)[..., 2:]
    caches = [torch.zeros((8, 3, 16, 64), dtype=dtype, device="cuda") for _ in range(4)]
    slots = dev(rng.permutation(128)[:100])
    args = dict(rotary_params=(c, s), positions=pos.reshape(2, 100), sections=(20, 11))
    got = afa.paged_append(rows, rows, *caches[:2], slots, q=rows, **args)
    rows = rows.contiguous()
    assert torch.equal(got, afa.paged_append(rows, rows, *caches[2:], slots, q=rows, **args))
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_of_single_entries_do_not_matter(dtype):
    """One token, one head, one batch row, one page: the stride of such an axis is never used, whatever it is."""
    rng = np.random.default_rng(16)
    c, s = tables(32, 16, F32)
    rows = dev(rng.standard_normal((3, 6 * 32 + 1)), dtype)[:, :192].unflatten(1, (6, 32))  # a projection of odd width
    q, k, v = rows[2:].split((4, 1, 1), 1)
    assert q.stride(0) % 2 == 1 and k.stride(0) % 2 == 1
    pos = dev([[3]])
    got = afa.apply_ago_rotations_axes(q, k, (c, s), pos, (16,))
    want = afa.apply_ago_rotations_axes(q.clone(), k.clone(), (c, s), pos, (16,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = dev(rng.standard_normal((1, 1, 5, 32)), dtype)
    odd = x.as_strided(x.shape, (331, 77, 32, 1))
    assert torch.equal(afa.apply_ago_rotations_axes(odd, None, (c, s), dev(np.arange(5)[None]), (16,))[0],
                       afa.apply_ago_rotations_axes(x, None, (c, s), dev(np.arange(5)[None]), (16,))[0])
    caches = [torch.zeros((1, 1, 16, 32), dtype=dtype, device="cuda") for _ in range(4)]
    views = [t.as_strided(t.shape, (1037, 519, 32, 1)) for t in caches[:2]]
    args = dict(q=q, rotary_params=(c, s), positions=pos, sections=(16,))
    assert torch.equal(afa.paged_append(k, v, *views, dev([7]), **args), want[0])
    afa.paged_append(k.clone(), v.clone(), *caches[2:], dev([7]))
    assert torch.equal(caches[0][0, 0, 7], want[1][0, 0]) and torch.equal(caches[1], caches[3])
    got = afa.afa_paged(q, *views, i32([[0]]), i32([8]), i32([0, 1]))
    assert torch.equal(got, afa.afa_paged(q.clone(), *caches[:2], i32([[0]]), i32([8]), i32([0, 1])))
    caches[0][0, 0, :8], caches[1][0, 0, :8] = (dev(rng.standard_normal((8, 32)), dtype) for _ in range(2))
    before = [t.clone() for t in caches[:2]]
    assert int(afa.paged_commit(*views, i32([[0]]), i32([2]), i32([8]), i32([[1, 3, -1]]))) == 4
    for t, b in zip(caches, before):
        assert torch.equal(t[0, 0, 2:4], b[0, 0, [3, 5]]) and torch.equal(t[0, 0, 4:], b[0, 0, 4:])


def test_tensors_written_in_place_say_so():
    """A backward pass that saved a tensor which one of the operators then changed is an error, not a wrong gradient."""
    rng = np.random.default_rng(18)
    caches = [dev(rng.standard_normal((4, 1, 16, 64)), F32) for _ in range(2)]
    k = dev(rng.standard_normal((3, 1, 64)), F32)
    table, free, one = i32([[0, 1, -1]]), i32([2, 3, 0]), i32([1])
    out = torch.zeros((1, 1, 64), device="cuda")
    path = i32([[1, 2]])
    calls = {
        "paged_append": (caches, lambda: afa.paged_append(k, k, *caches, dev([5, 6, 7]))),
        "paged_commit": (caches, lambda: afa.paged_commit(*caches, table, one, i32([8]), path)),
        "afa_paged": ([out], lambda: afa.afa_paged(k[:1], *caches, table, i32([8]), i32([0, 1]), out=out)),
        "paged_plan": ([table, free], lambda: afa.paged_plan(table, i32([2]), i32([8]), i32([40]), free, i32([2]), 16,
                                                             40)),
    }
    weight = torch.ones(8, device="cuda", requires_grad=True)
    for name, (written, call) in calls.items():
        for t in written:
            y = (weight[0] * t).sum()
            version = t._version
            with torch.no_grad():
                call()
            assert t._version > version, name
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    with torch.inference_mode():
        inside = [torch.zeros((4, 1, 16, 64), device="cuda") for _ in range(2)]
        afa.paged_append(k, k, *inside, dev([5, 6, 7]))
    afa.paged_append(k, k, *inside, dev([5, 6, 7]))


def exact(b, sink=0.5):
    """(out, d_total, sum p |v| / d_total) of a Batch in float64, request by request, on the GPU."""
    q, k, v, table, lens, cu, words = b.args()
    group, page, dim = q.shape[1] // k.shape[1], k.shape[2], q.shape[2]
    outs, dens, mags = [], [], []
    for i, (n, length) in enumerate(zip(b.new.tolist(), b.lens.tolist())):
        at = slice(int(b.cu[i]), int(b.cu[i]) + n)
        pages = table[i, :-(-length // page)].long()
        kk, vv = (x[pages].transpose(1, 2).reshape(-1, *x.shape[1::2])[:length].double().repeat_interleave(group, 1)
                  for x in (k, v))
        x = torch.einsum("nhd,lhd->nhl", q[at].double(), kk) / np.sqrt(dim)
        node = torch.arange(length, device="cuda") - (length - n)
        if words is None:
            seen = node[None] <= torch.arange(n, device="cuda")[:, None]
        else:
            w = torch.nn.functional.pad(words[at].long(), (0, 9))[:, (node >> 5).clamp(min=0)]
            seen = (node < 0)[None] | ((w >> (node & 31)) & 1).bool()
        p = torch.exp(8 * torch.asinh(x)) * seen[:, None]
        den = p.sum(-1) + sink
        dens.append(den)
        outs.append(torch.einsum("nhl,lhd->nhd", p, vv) / den[..., None])
        mags.append(torch.einsum("nhl,lhd->nhd", p, vv.abs()) / den[..., None])
    return torch.cat(outs), torch.cat(dens), torch.cat(mags)


def check_exactly(b, weight, sink=0.5, **kw):
    """Outputs within half a step of their type, and `weight` of sum p |v| for what the weights are off."""
    got, gden = afa.afa_paged(*b.args(), sink_omega=sink, return_denominator=True, **kw)
    assert _lib.device_status(got.device) == 0
    want, den, mag = exact(b, sink)
    t = want.shape[0]
    half = torch.maximum(want.abs(), got[:t].double().abs()).log2().floor().exp2() * torch.finfo(got.dtype).eps / 2
    off = ((got[:t].double() - want).abs() - half) / mag
    assert off.max().item() <= weight
    assert ((gden[:t].double() - den).abs() / den).max().item() <= min(weight, 3e-4)


# What a weight is off in the tensor-core kernels, without its own rounding. The score: products of bfloat16 are
# exact, their sum of at most 128 is off by sqrt(128) 2^-23 sum |q k| (under 110 for unit-normal numbers) / sqrt(128), and
# rho^8 takes eight times that: 1.1e-4. The map: 2.5e-6 s^2, under 6e-5 for these scores. Two bfloat16 parts: 2^-17.
# Together under 1.8e-4, bound 3e-4; a single bfloat16 weight adds half a step, 2^-8.
SPLIT, SINGLE = 3e-4, 3e-4 + 2.0 ** -8


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 7, 16])
def test_attention_rows_of_few_keys(dim, group):
    """Where roundings of single weights do not average out: requests of one to four keys, and trees on them. The
    transposed kernel holds weights in two parts; the row-tile kernel, for 40 tokens a request, in one."""
    lens = [1, 2, 3, 4] * 12
    check_exactly(Batch(19, [1] * 48, lens, 2, group, dim, 16, BF), SPLIT)
    two = 2 if group <= 16 else 1
    check_exactly(Batch(20, [two] * 48, [x + two for x in lens], 2, group, dim, 16, BF, tree=True), SPLIT)
    check_exactly(Batch(21, [40] * 6, [40, 41, 42, 43, 44, 40], 2, group, dim, 16, BF, tree=True), SINGLE)
    check_exactly(Batch(22, [40] * 6, [40, 41, 42, 43, 44, 40], 2, group, dim, 16, BF), SINGLE)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 7])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_mixed_batch_in_64_bits(dim, group, tree):
    """Single tokens, trees and chunks in one batch, and short and long requests of few rows, each row by itself."""
    rng = np.random.default_rng(23)
    new = rng.choice([1, 2, 7, 31, 33, 64, 65, 120, 200], 40)
    check_exactly(Batch(24, new, new + rng.integers(0, 900, 40), 2, group, dim, 32, BF, tree=tree), SINGLE)
    few = rng.choice([1, 1, 1, 2, 3], 60)
    lens = np.where(rng.random(60) < 0.2, rng.integers(3, 5000, 60), rng.integers(3, 300, 60))
    check_exactly(Batch(25, few, lens, 2, group, dim, 64, BF, tree=tree), SPLIT)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,group", [(1, 4), (8, 4)])
def test_attention_pieces_of_every_length_in_64_bits(dim, new, group):
    lens = [max(new, 128 * (i % 9) + 1 + 37 * i % 128) for i in range(60)]
    check_exactly(Batch(26, [new] * 60, lens, 3, group, dim, 128, BF), SPLIT)


@pytest.mark.parametrize("dtype,weight", [(F32, 1e-5), (F64, 1e-13)])
def test_attention_mixed_batch_on_cuda_cores_in_64_bits(dtype, weight):
    """float32: the bound at the head of this file (a score is off by about 7e-7, its weight by eight times that: 5e-6,
    bound 1e-5), here of each row's sum p |v| and not of the largest output. float64 2^-29 of that on either side:
    4e-14, bound 1e-13."""
    rng = np.random.default_rng(27)
    new = rng.choice([1, 2, 7, 31, 33, 64], 20)
    for dim in (64, 100, 128):
        check_exactly(Batch(28, new, new + rng.integers(0, 600, 20), 2, 5, dim, 32, dtype, tree=True), weight)


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (BF, 64), (F32, 64)])
@pytest.mark.parametrize("name", ["decode", "odd-group", "chunk", "tree", "wide-tree", "long-tree"])
def test_attention_into_its_queries(name, dtype, dim):
    """A unit's rows are read before they are written, and by no other unit."""
    b = Batch(29, dim=dim, dtype=dtype, **CASES[name])
    want = afa.afa_paged(*b.args())
    for _ in range(3):
        q, *rest = b.args()
        q = q.clone()
        assert afa.afa_paged(q, *rest, out=q) is q
        assert torch.equal(q, want)


def test_rotation_of_one_input_that_wants_a_gradient():
    """The other's result wants none, and both have the bits of a rotation together."""
    rng = np.random.default_rng(30)
    c, s = tables(32, 16, F32)
    pos, up = dev(rng.integers(0, 16, (2, 1, 7))), dev(rng.standard_normal((1, 4, 7, 32)), F32)
    x, y = (dev(rng.standard_normal((1, h, 7, 32)), F32) for h in (4, 2))
    want = afa.apply_ago_rotations_axes(x, y, (c, s), pos, (7, 9))
    back, = torch.autograd.grad(afa.apply_ago_rotations_axes(x.requires_grad_(True), None, (c, s), pos, (7, 9))[0], x, up)
    qr, kr = afa.apply_ago_rotations_axes(x, y, (c, s), pos, (7, 9))
    assert qr.requires_grad and not kr.requires_grad and torch.equal(qr, want[0]) and torch.equal(kr, want[1])
    assert torch.equal(torch.autograd.grad(qr, x, up)[0], back)
    kr, qr = afa.apply_ago_rotations_axes(y, x, (c, s), pos, (7, 9))
    assert qr.requires_grad and not kr.requires_grad and torch.equal(torch.autograd.grad(qr, x, up)[0], back)
