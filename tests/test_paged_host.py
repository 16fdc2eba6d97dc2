"""Refusals of the paged-cache operators and of the rotation with several axes, found before any CUDA call."""
import ctypes

import numpy as np
import pytest
import torch

import algebraic_intelligence_b200 as afa
from algebraic_intelligence_b200 import _lib
from algebraic_intelligence_b200.ago import axis_arguments
from oracle import paged_oracle as po

I32 = torch.int32


def _z(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def _plan(**change):
    args = dict(block_table=_z(2, 4), page_counts=_z(2), seq_lens=_z(2), new_lens=_z(2), free_pages=_z(8),
                free_count=_z(1), page_size=16, max_tokens=4)
    return afa.paged_plan(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    ({"block_table": _z(2, 4, dtype=torch.int64)}, TypeError),
    ({"block_table": _z(4, 2).t()}, ValueError),
    ({"block_table": _z(2, 0)}, ValueError),
    ({"page_counts": _z(3)}, ValueError),
    ({"seq_lens": _z(2, dtype=torch.int64)}, TypeError),
    ({"free_count": _z(2)}, ValueError),
    ({"free_pages": _z(0)}, ValueError),
    ({"page_size": 48}, ValueError),
    ({"page_size": 8}, ValueError),
    ({"page_size": 512}, ValueError),
    ({"max_tokens": -1}, ValueError),
    ({"max_tokens": 2 ** 30 + 1}, ValueError),
    ({"parents": _z(2, 257)}, ValueError),
    ({"parents": _z(3, 4)}, ValueError),
    ({}, ValueError),  # CPU tensors
])
def test_plan_refusals(change, error):
    with pytest.raises(error):
        _plan(**change)


def _attend(**change):
    bf = torch.bfloat16
    args = dict(q=_z(3, 4, 64, dtype=bf), k_cache=_z(5, 2, 16, 64, dtype=bf), v_cache=_z(5, 2, 16, 64, dtype=bf),
                block_table=_z(2, 3), seq_lens=_z(2), cu_tokens=_z(3))
    return afa.afa_paged(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    ({"q": _z(3, 3, 64, dtype=torch.bfloat16)}, ValueError),
    ({"q": _z(3, 4, 32, dtype=torch.bfloat16)}, ValueError),
    ({"q": _z(3, 4, 64, dtype=torch.float32)}, TypeError),
    ({"q": _z(3, 4, 64)}, TypeError),
    ({k: _z(*s, dtype=torch.float16) for k, s in (("q", (3, 4, 64)), ("k_cache", (5, 2, 16, 64)),
                                                  ("v_cache", (5, 2, 16, 64)))}, TypeError),
    ({"v_cache": _z(5, 2, 32, 64, dtype=torch.bfloat16)}, ValueError),
    ({"k_cache": _z(5, 2, 24, 64, dtype=torch.bfloat16), "v_cache": _z(5, 2, 24, 64, dtype=torch.bfloat16)},
     ValueError),
    ({"k_cache": _z(5, 2, 64, 16, dtype=torch.bfloat16).mT}, ValueError),
    ({"block_table": _z(2, 3, dtype=torch.int64)}, TypeError),
    ({"seq_lens": _z(3)}, ValueError),
    ({"cu_tokens": _z(2)}, ValueError),
    ({"ancestors": _z(2, 1)}, ValueError),
    ({"ancestors": _z(3, 1, dtype=torch.int64)}, TypeError),
    ({"sink_omega": -1.0}, ValueError),
    ({"sink_omega": float("nan")}, ValueError),
    ({"out": _z(3, 4, 64, dtype=torch.float32)}, ValueError),
    ({"q": _z(3, 4, 64, dtype=torch.bfloat16).requires_grad_(True)}, ValueError),
    ({}, ValueError),  # CPU tensors
])
def test_attention_refusals(change, error):
    with pytest.raises(error):
        _attend(**change)


def _append(**change):
    f = torch.float32
    args = dict(k=_z(3, 2, 8, dtype=f), v=_z(3, 2, 8, dtype=f), k_cache=_z(5, 2, 16, 8, dtype=f),
                v_cache=_z(5, 2, 16, 8, dtype=f), slots=_z(3, dtype=torch.int64))
    return afa.paged_append(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    ({"k": _z(3, 2, 6, dtype=torch.float32)}, ValueError),
    ({"v": _z(2, 2, 8, dtype=torch.float32)}, ValueError),
    ({"k": _z(3, 2, 8, dtype=torch.float64)}, TypeError),
    ({"slots": _z(2, dtype=torch.int64)}, ValueError),
    ({"slots": _z(3, dtype=torch.float32)}, TypeError),
    ({"q": _z(3, 4, 8, dtype=torch.float32)}, ValueError),  # q without tables
    ({"q": _z(4, 4, 8, dtype=torch.float32)}, ValueError),
    ({"positions": _z(1, 3)}, ValueError),
    ({"k": _z(3, 2, 8, dtype=torch.float32).requires_grad_(True)}, ValueError),
    ({"k_cache": _z(5, 2, 16, 8, dtype=torch.float32).requires_grad_(True)}, ValueError),
    ({}, ValueError),  # CPU tensors
])
def test_append_refusals(change, error):
    with pytest.raises(error):
        _append(**change)


def _commit(**change):
    f = torch.float32
    args = dict(k_cache=_z(5, 2, 16, 8, dtype=f), v_cache=_z(5, 2, 16, 8, dtype=f), block_table=_z(2, 3),
                base_lens=_z(2), seq_lens=_z(2), accepted=_z(2, 4))
    return afa.paged_commit(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    ({"accepted": _z(2, 257)}, ValueError),
    ({"accepted": _z(3, 4)}, ValueError),
    ({"accepted": _z(2, 4, dtype=torch.int64)}, TypeError),
    ({"base_lens": _z(3)}, ValueError),
    ({"block_table": _z(6)}, ValueError),
    ({"v_cache": _z(5, 2, 16, 8, dtype=torch.float32).requires_grad_(True)}, ValueError),
    ({"v_cache": _z(5, 2, 16, 6, dtype=torch.float32)}, ValueError),
    ({}, ValueError),  # CPU tensors
])
def test_commit_refusals(change, error):
    with pytest.raises(error):
        _commit(**change)


def _rotate(**change):
    x = np.zeros((2, 3, 5, 8))
    args = dict(q=x, k=x[:, :1], rotary_params=(np.ones((9, 4)), np.zeros((9, 4))),
                positions=np.zeros((2, 2, 5), np.int32), sections=(2, 1))
    return afa.apply_ago_rotations_axes(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    ({"q": np.zeros((2, 3, 5, 7))}, ValueError),
    ({"q": np.zeros((5, 8))}, ValueError),
    ({"k": np.zeros((2, 3, 4, 8))}, ValueError),
    ({"k": np.zeros((2, 0, 5, 8))}, ValueError),
    ({"q": np.zeros((2, 3, 5, 8), np.int32)}, TypeError),
    ({"sections": (3, 2)}, ValueError),
    ({"sections": (-1, 2)}, ValueError),
    ({"sections": (1, 1, 1, 1, 0)}, ValueError),
    ({"sections": (2,)}, ValueError),  # two axes of positions
    ({"sections": None}, ValueError),
    ({"positions": np.zeros((2, 2, 4), np.int32)}, ValueError),
    ({"positions": np.zeros((2, 2, 5))}, TypeError),
    ({"positions": np.full((2, 2, 5), 9)}, ValueError),
    ({"positions": np.full((2, 2, 5), -1)}, ValueError),
    ({"rotary_params": (np.ones((9, 5)), np.zeros((9, 5)))}, ValueError),
    ({"rotary_params": (np.ones((9, 4)), np.zeros((8, 4)))}, ValueError),
    ({"rotary_params": (np.ones((9, 4)), np.zeros((9, 4), np.float32))}, TypeError),
    ({"rotary_params": (torch.ones(9, 4).requires_grad_(True), torch.zeros(9, 4))}, ValueError),
    ({"q": torch.zeros(2, 3, 5, 8).requires_grad_(True), "k": None}, ValueError),
])
def test_rotation_refusals(change, error):
    with pytest.raises(error):
        _rotate(**change)


@pytest.mark.parametrize("shape", [(0, 2, 16, 64), (5, 0, 16, 64), (5, 2, 16, 0)])
def test_empty_caches_are_refused(shape):
    empty = dict(k_cache=torch.zeros(shape), v_cache=torch.zeros(shape))
    for call in (_attend, _append, _commit):
        with pytest.raises(ValueError, match="must not be empty"):
            call(**empty)


def test_out_that_wants_a_gradient_is_refused():
    with pytest.raises(ValueError, match="has no gradient"):
        _attend(out=_z(3, 4, 64, dtype=torch.bfloat16).requires_grad_(True))


def test_sections_are_integers():
    with pytest.raises(TypeError):
        _rotate(sections=(2.5, 1))
    # Read at every call, whatever holds them.
    sections = [torch.tensor(2), torch.tensor(1)]
    assert np.array_equal(axis_arguments((np.ones((9, 4)), np.zeros((9, 4))), np.zeros((2, 5), np.int32), sections, 8,
                                         (5,), None).sections[:2], [2, 1])
    sections[0].add_(1)
    assert np.array_equal(axis_arguments((np.ones((9, 4)), np.zeros((9, 4))), np.zeros((2, 5), np.int32), sections, 8,
                                         (5,), None).sections[:2], [3, 1])


def test_c_entries_refuse_before_any_cuda_call():
    lib = _lib.load()
    inv, dt = _lib.AFA_ERR_INVALID, _lib.AFA_ERR_DTYPE
    two, three = (ctypes.c_longlong * 2)(1, 1), (ctypes.c_longlong * 3)(1, 1, 1)
    four, secs = (ctypes.c_longlong * 4)(1, 1, 1, 1), (ctypes.c_int * 2)(2, 2)

    def attend(**c):
        a = dict(D=64, dtype=_lib.AFA_BF16, page=16, q_heads=4, sink=0.5, cols=3, words=0, anc=None, ws=1 << 40)
        a.update(c)
        return lib.afa_paged(16, two, 16, 16, three, three, 16, None, 16, 3, 16, 16, a["anc"], 1, a["words"], 1, 3,
                             a["q_heads"], 2, a["D"], a["cols"], a["page"], 5, a["dtype"], a["sink"], 16, a["ws"],
                             None)

    assert attend(dtype=_lib.AFA_F16) == dt and attend(dtype=9) == dt
    for bad in ({"D": 257}, {"D": 0}, {"page": 24}, {"page": 512}, {"q_heads": 3}, {"sink": -1.0},
                {"sink": float("inf")}, {"cols": 1 << 27}, {"anc": 16, "words": 0}, {"ws": 64}):
        assert attend(**bad) == inv, bad
    assert b"workspace" in lib.afa_last_error()
    assert lib.afa_paged_workspace_bytes(0, 4, 2, 64, _lib.AFA_BF16) == 0
    assert lib.afa_paged_workspace_bytes(3, 4, 2, 64, _lib.AFA_BF16) > 0

    def plan(batch=2, cols=4, page=16, free=8, nodes=0, parents=None):
        return lib.afa_paged_plan(*[16] * 6, parents, *[16] * 9, batch, cols, page, free, 4, nodes, None)

    for bad in ({"batch": 0}, {"batch": 4097}, {"cols": 0}, {"page": 20}, {"free": 0}, {"cols": 1 << 27},
                {"parents": 16, "nodes": 257}, {"parents": 16, "nodes": 0}):
        assert plan(**bad) == inv, bad

    def rotate(dim=8, dtype=_lib.AFA_F32, sections=secs, axes=2, q=16, strides=three):
        return lib.afa_ago_rotate_axes(q, strides, 16, 1, None, None, None, 0, 16, 16, _lib.AFA_F32, 4, 16, three, 0,
                                       sections, axes, 1, 1, 2, dim, 0, dtype, None)

    assert rotate(dtype=_lib.AFA_F16) == dt
    for bad in ({"dim": 7}, {"dim": 6}, {"axes": 0}, {"axes": 5}, {"q": None}, {"sections": None}):
        assert rotate(**bad) == inv, bad
    assert rotate() == inv and b"alignment" in lib.afa_last_error()  # strides of one element

    assert lib.afa_paged_append(16, two, 16, two, 16, three, 16, three, 16, 16, two, 16, 2, None, None, 0, 0, None,
                                None, 0, None, 0, 3, 2, 8, 5, 16, _lib.AFA_F32, None) == inv
    assert b"rotary" in lib.afa_last_error()
    assert lib.afa_paged_commit(16, four, 16, four, 16, 3, 16, 16, 16, 4, 16, 2, 300, 1, 2, 8, 3, 5, 16,
                                _lib.AFA_F32, None) == inv
    assert lib.afa_paged_commit(16, four, 16, four, 16, 3, 16, 16, 16, 4, 16, 2, 4, 1, 2, 8, 3, 5, 16,
                                _lib.AFA_F16, None) == dt


def test_oracle_plan_conserves_pages():
    """Pages held and pages on the stack partition the pool after any step."""
    rng = np.random.default_rng(0)
    table, held, lens = np.full((4, 6), -1, np.int32), np.zeros(4, int), np.zeros(4, int)
    stack, free = np.arange(12, dtype=np.int32), 12
    for _ in range(40):
        new = rng.integers(0, 40, 4)
        lens = np.where(rng.random(4) < 0.3, rng.integers(0, lens + 1), lens)
        r = po.plan(table, held, lens, new, stack, free, 16, 100)
        table, held, lens = r["block_table"], r["page_counts"].astype(int), r["seq_lens"].astype(int)
        stack, free = r["free_pages"], int(r["free_count"][0])
        pages = [table[b, j] for b in range(4) for j in range(held[b])] + list(stack[:free])
        assert sorted(pages) == list(range(12))


def test_oracle_causal_attention_is_the_dense_one():
    from oracle import afa_oracle as orc
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((21, h, 8)) for h in (4, 2, 2))
    table = np.array([[1, 0]])
    caches = []
    for x in (k, v):
        c = np.zeros((2, 2, 16, 8))
        c[1], c[0, :, :5] = x[:16].transpose(1, 0, 2), x[16:].transpose(1, 0, 2)
        caches.append(c)
    out, _ = po.attend(q, *caches, table, [21], [0, 21])
    dense = orc.afa(*(x.transpose(1, 0, 2)[None] for x in (q, k.repeat(2, 1), v.repeat(2, 1))), causal=True)
    assert np.max(np.abs(out.transpose(1, 0, 2)[None] - dense)) < 1e-13


def test_c_rotation_refuses_outputs_off_a_channel_pair():
    """The kernel stores a pair at a time: an output off one would be a misaligned access."""
    lib = _lib.load()
    three, secs = (ctypes.c_longlong * 3)(2, 2, 2), (ctypes.c_int * 1)(1)
    for dtype, size in ((_lib.AFA_BF16, 2), (_lib.AFA_F32, 4), (_lib.AFA_F64, 8)):
        for q_out, k_out in ((4096 + size, 4096), (4096, 4096 + size)):
            assert lib.afa_ago_rotate_axes(4096, three, q_out, 1, 4096, three, k_out, 1, 4096, 4096, _lib.AFA_F32, 4,
                                           4096, three, 0, secs, 1, 1, 1, 2, 2, 0, dtype, None) == _lib.AFA_ERR_INVALID
            assert b"alignment" in lib.afa_last_error()


def test_forward_mode_tangents_are_refused():
    """Not dropped: also of tensors that want no gradient, and where no gradients are recorded."""
    from torch.autograd import forward_ad as fw
    f = torch.float32

    def dual(*shape):
        return fw.make_dual(_z(*shape, dtype=f), torch.ones(shape))

    x = torch.zeros(2, 3, 5, 8)
    tables = torch.ones(9, 4), torch.zeros(9, 4)
    cache, q = _z(5, 2, 16, 64, dtype=f), _z(3, 4, 64, dtype=f)
    with fw.dual_level(), torch.no_grad():
        for call in (lambda: _rotate(q=dual(2, 3, 5, 8), k=x[:, :1]), lambda: _rotate(q=x, k=dual(2, 1, 5, 8)),
                     lambda: _rotate(q=x, k=None, rotary_params=(dual(9, 4), tables[1])),
                     lambda: _append(k=dual(3, 2, 8)), lambda: _append(v_cache=dual(5, 2, 16, 8)),
                     lambda: _commit(k_cache=dual(5, 2, 16, 8)),
                     lambda: _attend(q=dual(3, 4, 64), k_cache=cache, v_cache=cache),
                     lambda: _attend(q=q, k_cache=cache, v_cache=dual(5, 2, 16, 64))):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call()


@pytest.mark.parametrize("layers", [0, 2])
def test_caches_whose_rows_share_memory_are_refused(layers, monkeypatch):
    """They are written to. Ordinary views, also both caches in one buffer, are not (here they get as far as the
    launch, with tensors that only claim to be on a GPU)."""
    from algebraic_intelligence_b200 import paged
    monkeypatch.setattr(paged, "_one_device", lambda *tensors: torch.device("cpu"))

    class Launched(Exception):
        pass

    def launch(*args):
        raise Launched

    monkeypatch.setattr(_lib, "call", launch)
    f, lead = torch.float32, (layers,) if layers else ()
    z = lambda *shape: _z(*lead, *shape, dtype=f)  # noqa: E731
    calls = [_commit] if layers else [_commit, _append]
    plain = z(5, 2, 16, 8)
    wide = z(5, 2, 2, 16, 8)
    fused, pool, far = z(5, 16, 2, 24), z(10, 2, 16, 8), z(18, 2, 16, 8)
    for k, v in ((plain, z(5, 2, 16, 8)), (z(5, 16, 2, 8).transpose(-3, -2), z(5, 16, 2, 8).transpose(-3, -2)),
                 (z(5, 16, 2, 8).transpose(-3, -2), plain), (wide.select(-4, 0), wide.select(-4, 1)),
                 (wide.select(-4, 1), wide.select(-4, 0)), (wide.select(-3, 0), wide.select(-3, 1)),
                 (fused[..., :8].transpose(-3, -2), fused[..., 16:].transpose(-3, -2)),
                 (pool[..., ::2, :, :, :], pool[..., 1::2, :, :, :]), (pool[..., 5:, :, :, :], pool[..., :5, :, :, :]),
                 (far[..., :10:2, :, :, :], far[..., 5:15:2, :, :, :]), (far[..., 9::2, :, :, :], far[..., :10:2, :, :, :])):
        for call in calls:
            with pytest.raises(Launched):
                call(k_cache=k, v_cache=v)
    spread = z(5, 1, 16, 8).expand(*lead, 5, 2, 16, 8)
    pages = z(1, 2, 16, 8).expand(*lead, 5, 2, 16, 8)
    window = torch.zeros(4000).as_strided((*lead, 5, 2, 16, 8), (*(2000,) * len(lead), 256, 128, 4, 1))
    for k, v in ((spread, plain), (plain, pages), (plain, plain), (plain, window), (window, window),
                 (wide.select(-4, 0), wide.select(-4, 0)), (spread, spread), (pool[..., :5, :, :, :], pool[..., 4:9, :, :, :]),
                 (far[..., :10:2, :, :, :], far[..., 4:14:2, :, :, :])):
        for call in calls:
            with pytest.raises(ValueError, match="share memory"):
                call(k_cache=k, v_cache=v)
