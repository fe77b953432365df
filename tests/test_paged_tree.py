"""Drafted trees, parts of prompts and shared pages over a paged cache
(pcl_page_tree_masks, pcl_page_accept, pcl_page_fork, pcl_page_release_shared,
pcl_paged_copy, pcl_paged_tree_attention).

Bookkeeping is checked word for word against models that handle one request, token
or page after another; copies bit for bit; attention bit for bit against
pcl_attention_launch over each request's rows in one segment with the same keys
seen, and against a softmax in 64 bits. The runs at the end take a batch through
rounds of drafted trees and through forks, beside the same tokens decoded one at a
time.
"""
import ctypes

import numpy as np
import pytest

import test_paged as tp
from test_paged import (BAD_PAGES, STATE, Cache, DeviceBatch, PageModel, Pools, batch_of, bits,
                        ctx, no_context, pools_of, scale_of, torch)  # noqa: F401


# ---- models ------------------------------------------------------------------

class ShareModel(PageModel):
    """The bookkeeping with forks and shared pages."""

    def fork(self, sources):
        """(from, to, rows) or None when it is refused."""
        self.void()
        self.standing = None
        made = []
        for b, s in enumerate(sources):
            if s < 0:
                continue
            if s >= self.requests or self.lengths[b] or sources[s] >= 0:
                return None
            if self.lengths[s] % self.page:
                made.append(b)
        if len(made) > len(self.free):
            return None
        out = [[-1] * self.requests, [-1] * self.requests, [0] * self.requests]
        for b, s in enumerate(sources):
            if s < 0:
                continue
            n = self.lengths[s]
            whole = n // self.page
            self.table[b][:whole] = self.table[s][:whole]
            if n % self.page:
                fresh = self.free[len(self.free) - 1 - self.taken]
                self.taken += 1
                self.table[b][whole] = fresh
                out[0][b], out[1][b] = self.table[s][whole] * self.page, fresh * self.page
                out[2][b] = n % self.page
            self.step_lengths[b] = n
        self.standing = [self.step_lengths[b] - self.lengths[b] for b in range(self.requests)]
        self.state = 2
        return out

    def step(self, counts):
        self.state = 1
        return super().step(counts)

    state = 1

    def check(self, state):
        standing, self.standing = self.standing, None
        state = dict(state, counters=state["counters"].copy())
        assert state["counters"][3] == (self.state if standing is not None else 0)
        state["counters"][3] = 0
        super().check(state)
        self.standing = standing

    def pages_of(self, b):
        return self.table[b][:self.held(self.lengths[b])]

    def release_shared(self, finished):
        kept = {p for b in range(self.requests) if not finished[b] for p in self.pages_of(b)}
        gone = {p for b in range(self.requests) if finished[b] for p in self.pages_of(b)}
        self.free += sorted(gone - kept, reverse=True)
        self.lengths = [0 if f else n for n, f in zip(self.lengths, finished)]
        self.standing = None


def tree_of(parents):
    """(depth, branches) of one request's new tokens."""
    depth, branch = [], []
    for i, p in enumerate(parents):
        depth.append(depth[p] + 1 if p >= 0 else 0)
        branch.append((branch[p] if p >= 0 else set()) | {i})
    return depth, branch


def words_of(branch, words):
    """A set of token indexes as signed 64-bit words."""
    bits_ = np.zeros(words * 64, np.uint8)
    bits_[list(branch)] = 1
    return np.packbits(bits_, bitorder="little").view(np.int64)


def random_parents(rng, n):
    kind = rng.integers(4)
    if kind == 0:
        return [i - 1 for i in range(n)]
    if kind == 1:
        return [-1] * n
    return [int(rng.integers(max(-1, i - 5) if kind == 2 else -1, i)) for i in range(n)]


def test_the_models_themselves():
    m = ShareModel(4, 4, 4, 8, 32)
    assert m.step([6, 4, 0, 0]) and m.commit()
    assert m.fork([-1, -1, 0, 2]) is None  # the source is a fork
    assert m.fork([-1, 0, -1, -1]) is None  # holds tokens
    assert m.fork([-1, -1, 4, -1]) is None
    assert m.fork([-1, -1, 0, 1]) == [[-1, -1, 4, -1], [-1, -1, 12, -1], [0, 0, 2, 0]]
    assert m.commit() and m.lengths == [6, 4, 6, 4] and m.free == [7, 6, 5, 4]
    assert m.table[2][:2] == [0, 3] and m.table[3][:1] == [2]
    m.release_shared([1, 0, 0, 0])
    assert m.free == [7, 6, 5, 4, 1]
    m.release_shared([0, 1, 0, 1])
    assert m.free == [7, 6, 5, 4, 1, 2]
    m.release_shared([0, 0, 1, 0])
    assert sorted(m.free) == list(range(8))
    depth, branch = tree_of([-1, 0, 0, 1, -1])
    assert depth == [0, 1, 1, 2, 0] and branch[3] == {0, 1, 3} and branch[4] == {4}
    assert words_of({0, 63, 64}, 2).view(np.uint64).tolist() == [1 | 1 << 63, 1]


# ---- refusals (no device work) ----------------------------------------------

def tree_desc_of(pcl, pools=None, **kw):
    fields = dict(q=64, q_stride=256, q_rows=8, qheads=4, table=64, table_stride=4, lengths=64,
                  step_lengths=64, newest=64, requests=2, max_length=64, max_new=4, out=64,
                  o_stride=256)
    fields.update(kw)
    return pcl.Context.paged_tree_desc(pools=pools or pools_of(pcl), **fields)


@pytest.mark.parametrize("kw", [dict(requests=0), dict(requests=2049), dict(page_tokens=4097),
                                dict(pages=0), dict(step_rows=1 << 20)] +
                         [{n: None} for n in STATE] + [{n: 66} for n in STATE], ids=str)
def test_page_calls_refuse_bad_batches(pcl, no_context, kw):
    lib = pcl.load()
    b = ctypes.byref(batch_of(pcl, **kw))
    w = ctypes.c_void_p(64)
    t = ctypes.byref(pcl.page_tree(parents=64, words=1, positions=64, masks=64))
    assert lib.pcl_page_tree_masks(no_context, b, t) == pcl.INVALID_SHAPE
    assert lib.pcl_page_accept(no_context, b, w, w, 4, w, w) == pcl.INVALID_SHAPE
    assert lib.pcl_page_fork(no_context, b, w, w, w, w) == pcl.INVALID_SHAPE
    assert lib.pcl_page_release_shared(no_context, b, w) == pcl.INVALID_SHAPE
    assert lib.pcl_page_release_workspace_bytes(b) == 0


@pytest.mark.parametrize("kw", [dict(parents=None), dict(parents=66), dict(words=0),
                                dict(words=9), dict(words=-1), dict(positions=None),
                                dict(positions=65), dict(masks=None), dict(masks=68)], ids=str)
def test_trees_refuse_bad_arrays(pcl, no_context, kw):
    lib = pcl.load()
    fields = dict(parents=64, words=2, positions=64, masks=64)
    fields.update(kw)
    b = ctypes.byref(batch_of(pcl))
    assert lib.pcl_page_tree_masks(no_context, b, ctypes.byref(pcl.page_tree(**fields))) == \
        pcl.INVALID_SHAPE
    assert lib.pcl_page_tree_masks(no_context, b, None) == pcl.INVALID_SHAPE
    assert lib.pcl_page_tree_masks(None, b, ctypes.byref(pcl.page_tree())) == pcl.INVALID_SHAPE


def test_page_calls_refuse_missing_words(pcl, no_context):
    lib = pcl.load()
    b = ctypes.byref(batch_of(pcl))
    w = ctypes.c_void_p(64)
    for i in range(4):
        for bad in (None, ctypes.c_void_p(66)):
            p = [bad if i == j else w for j in range(4)]
            assert lib.pcl_page_accept(no_context, b, p[0], p[1], 4, p[2], p[3]) == 1
            assert lib.pcl_page_fork(no_context, b, *p) == 1
    for depth in (0, -1, 1 << 20, 1 << 40):
        assert lib.pcl_page_accept(no_context, b, w, w, depth, w, w) == 1
    for bad in (None, ctypes.c_void_p(66)):
        assert lib.pcl_page_release_shared(no_context, b, bad) == 1
    assert lib.pcl_page_accept(None, b, w, w, 4, w, w) == 1
    assert lib.pcl_page_fork(None, b, w, w, w, w) == 1
    assert lib.pcl_page_release_shared(None, b, w) == 1
    assert lib.pcl_page_release_workspace_bytes(None) == 0
    # two bytes a page in whole 32, none for a small batch
    def nbytes(**kw):
        return lib.pcl_page_release_workspace_bytes(ctypes.byref(batch_of(pcl, **kw)))
    assert nbytes() == nbytes(table_stride=1 << 13) == nbytes(pages=1 << 17) == 0
    wide = nbytes(table_stride=1 + (1 << 13), pages=65)
    assert wide >= 2 * 96 + 16
    assert nbytes(pages=1 + (1 << 17)) - wide == 2 * (32 + (1 << 17) - 96)


def test_copy_refuses_bad_lists(pcl, no_context):
    lib = pcl.load()
    p = ctypes.c_void_p(64)

    def call(pools, *args, layers=None):
        array = (pcl.PclPagePools * max(1, len(pools)))(*pools)
        return lib.pcl_paged_copy(no_context, array, len(pools) if layers is None else layers,
                                  *args)

    good = pools_of(pcl)
    for kw in tp.BAD_POOLS:
        assert call([good, pools_of(pcl, **kw)], p, p, None, 1, 1) == 1, kw
    for other in (dict(pages=9), dict(page_tokens=8)):  # the layers' pages differ
        assert call([good, pools_of(pcl, **other)], p, p, None, 1, 1) == 1
    odd = ctypes.c_void_p(66)
    for args in ((None, p, None, 1, 1), (p, None, None, 1, 1), (odd, p, None, 1, 1),
                 (p, odd, None, 1, 1), (p, p, odd, 1, 1), (p, p, p, 1, 2), (p, p, None, -1, 1),
                 (p, p, None, 1, -1), (p, p, None, 1 << 20, 1), (p, p, None, 1, 1 << 20),
                 (p, p, None, (1 << 20) - 1, (1 << 20) - 1)):
        assert call([good], *args) == 1, args
    assert call([good], p, p, None, 1, 1, layers=-1) == 1
    assert call([good], p, p, None, 1, 1, layers=4097) == 1
    assert lib.pcl_paged_copy(no_context, None, 1, p, p, None, 1, 1) == 1
    assert lib.pcl_paged_copy(None, ctypes.byref(good), 1, p, p, None, 1, 1) == 1
    # nothing to do
    for args in ((None, None, None, 0, 1), (None, None, None, 1, 0)):
        assert call([good], *args) == pcl.OK
    assert call([], None, None, None, 1, 1) == pcl.OK


@pytest.mark.parametrize("kw,code", [
    (dict(qheads=0), 1), (dict(qheads=3), 1), (dict(qheads=4098), 1), (dict(requests=-1), 1),
    (dict(requests=2049), 1), (dict(window=-1), 1), (dict(q=None), 1), (dict(out=None), 1),
    (dict(table=None), 1), (dict(lengths=None), 1), (dict(step_lengths=None), 1),
    (dict(newest=None), 1), (dict(table_stride=0), 1), (dict(max_length=0), 1),
    (dict(max_length=65), 1), (dict(max_new=0), 1), (dict(max_new=1 << 20), 1),
    (dict(q_rows=0), 1), (dict(q_rows=1 << 20), 1), (dict(q_stride=252), 1),
    (dict(q_stride=258), 1), (dict(o_stride=252), 1), (dict(o_stride=257), 1), (dict(q=72), 1),
    (dict(out=72), 1), (dict(table=66), 1), (dict(lengths=66), 1), (dict(step_lengths=65), 1),
    (dict(newest=66), 1), (dict(mask_words=1), 1), (dict(positions=64), 1),
    (dict(masks=64), 1), (dict(masks=64, mask_words=9), 1), (dict(masks=68, mask_words=1), 1),
    (dict(masks=64, mask_words=1, window=5), 1),
    (dict(masks=64, mask_words=1, positions=66), 1), (dict(softcap=-1.0), 2),
    (dict(softcap=float("nan")), 2), (dict(softcap=float("inf")), 2), (dict(softcap=1e-40), 2),
    (dict(q_scale=float("nan")), 2), (dict(q_scale=float("inf")), 2),
    (dict(q_rows=1 << 19, max_length=1 << 30, table_stride=1 << 30), 1)], ids=str)
def test_attention_refuses_bad_descriptors(pcl, no_context, kw, code):
    lib = pcl.load()
    d = tree_desc_of(pcl, **kw)
    assert lib.pcl_paged_tree_attention(no_context, ctypes.byref(d)) == code
    assert lib.pcl_paged_tree_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.pcl_paged_tree_attention(None, ctypes.byref(tree_desc_of(pcl))) == 1
    assert lib.pcl_paged_tree_attention(no_context, None) == 1


@pytest.mark.parametrize("kw", tp.BAD_POOLS, ids=str)
def test_attention_refuses_bad_pools(pcl, no_context, kw):
    lib = pcl.load()
    d = tree_desc_of(pcl, pools_of(pcl, **kw))
    assert lib.pcl_paged_tree_attention(no_context, ctypes.byref(d)) == 1
    assert lib.pcl_paged_tree_workspace_bytes(ctypes.byref(d)) == 0


def test_workspace_holds_every_chunk_of_every_row(pcl):
    lib = pcl.load()

    def nbytes(**kw):
        return lib.pcl_paged_tree_workspace_bytes(ctypes.byref(tree_desc_of(
            pcl, pools_of(pcl, page_tokens=256, pages=64), table_stride=64, **kw)))

    part = 4 * 66 * 4  # (dim + 2) floats per query head
    base = nbytes(max_length=256)
    assert nbytes(max_length=1) == base > 0
    assert nbytes(max_length=257) - base == 8 * 2 * part
    assert nbytes(max_length=2561) - base == 8 * 11 * part
    assert nbytes(max_length=2561, q_rows=100) - base == 100 * 11 * part
    # a window's keys and the new tokens behind them: window + max_new - 1 keys lie
    # in at most (keys + 254) div 256 + 1 chunks
    assert nbytes(max_length=16384, window=1, max_new=1) == base
    assert nbytes(max_length=16384, window=1, max_new=2) - base == 8 * 2 * part
    assert nbytes(max_length=16384, window=1022, max_new=4) - base == 8 * 5 * part
    assert nbytes(max_length=16384, window=1023, max_new=4) - base == 8 * 6 * part
    assert nbytes(max_length=1000, window=(1 << 63) - 1, max_new=4) - base == 8 * 4 * part

    def plan(chunks):
        # above eight rows of a KV head: 64 bytes, and for each chunk, KV head and unit
        # of sixteen rows (16 in all, and one that every request ends in); 16 for the
        # requests' words
        return 64 * (1 + chunks * 2 * (16 // 16 + 2)) + 16

    assert nbytes(max_length=16384, window=1021, max_new=5) - base == 8 * 5 * part + plan(5)
    assert nbytes(max_length=16384, window=1022, max_new=258) - base == 8 * 6 * part + plan(6)
    assert nbytes(max_length=200, max_new=258) - base == plan(1)
    assert nbytes(requests=0) == 0


@pytest.mark.parametrize("source,kernel", [
    ("paged_tree_d256.hip", "_ZN3pcl17paged_tree_kernelILi256EfLb1ELi1ELi1EEEvNS_10TreeParamsE"),
    ("paged_rows_d256.hip", "_ZN3pcl16tree_rows_kernelILi256EfLb1ELi1ELi1EEEvNS_10TreeParamsE"),
    ("paged_rows_d256.hip", "_ZN3pcl16tree_rows_kernelILi256EDF16bLb1ELi1ELi1EEEvNS_10TreeParamsE"),
    ("paged_rows_d256.hip", "_ZN3pcl16tree_rows_kernelILi256EfLb1ELi3ELi1EEEvNS_10TreeParamsE"),
    ("paged_rows_d256.hip", "_ZN3pcl16tree_rows_kernelILi256EDF16bLb1ELi3ELi1EEEvNS_10TreeParamsE"),
    ("paged_rows_d512.hip", "_ZN3pcl16tree_rows_kernelILi512EfLb1ELi2ELi1EEEvNS_10TreeParamsE"),
    ("paged_tree.hip",
     "_ZN3pcl19tree_combine_kernelILi8EEEvNS_10TreeParamsENS_12CombineShapeE"),
])
def test_tree_kernels_do_not_spill_registers(source, kernel):
    import os
    from test_boundary import _resource_remarks
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc absent")
    spills = _resource_remarks(source)
    assert kernel in spills, sorted(spills)
    assert spills[kernel] == 0


# ---- trees on the device -------------------------------------------------------

class Trees:
    """A batch with a standing step and arrays for its trees."""

    def __init__(self, pcl, torch, ctx, shape, words):
        self.pcl, self.torch, self.ctx, self.words = pcl, torch, ctx, words
        self.batch = DeviceBatch(pcl, torch, *shape)
        self.rows = shape[4]
        dev = {"device": "cuda:0"}
        self.parents = torch.full((self.rows,), 5, dtype=torch.int32, **dev)
        self.positions = torch.full((self.rows,), 77, dtype=torch.int32, **dev)
        self.masks = torch.full((self.rows, words), 77, dtype=torch.int64, **dev)
        self.tree = pcl.page_tree(parents=self.parents.data_ptr(), words=words,
                                  positions=self.positions.data_ptr(),
                                  masks=self.masks.data_ptr())

    def put(self, parents):
        flat = [p for x in parents for p in x]
        self.parents.fill_(5)
        self.parents[:len(flat)] = self.torch.tensor(flat, dtype=self.torch.int32)

    def call(self):
        self.ctx.page_tree(self.batch.desc, self.tree)
        error = self.ctx.sync()
        return error, self.positions.cpu().numpy(), self.masks.cpu().numpy()


def expected(model, parents, rows, words):
    positions, masks = np.full(rows, -1), np.zeros((rows, words), np.int64)
    at = 0
    for held, mine in zip(model.lengths, parents):
        depth, branch = tree_of(mine)
        for d, b in zip(depth, branch):
            positions[at], masks[at] = held + d, words_of(b, words)
            at += 1
    return positions, masks


@pytest.mark.gpu
@pytest.mark.parametrize("words", [1, 2, 3, 8])
def test_masks_and_positions_follow_the_model(pcl, torch, ctx, words):
    shape = (7, 60, 16, 500, 2300)
    rng = np.random.default_rng(words)
    trees = Trees(pcl, torch, ctx, shape, words)
    model = ShareModel(*shape)
    call = tp.device_call(ctx, trees.batch)
    ctx.page_reset(trees.batch.desc)
    most = 64 * words
    for counts in ([5, 0, 1, 40, 0, 3, 7], [1, 1, 1, 1, 1, 1, 1], [0] * 7,
                   [most, 0, most - 1, 1, 64, 63, 2], [17, 33, 9, 0, 30, 1, 64]):
        assert model.step(counts) and call("step", counts)[0] == 0
        parents = [random_parents(rng, n) for n in counts]
        trees.put(parents)
        error, positions, masks = trees.call()
        assert error == 0
        want = expected(model, parents, shape[4], words)
        assert np.array_equal(positions, want[0]) and np.array_equal(masks, want[1])
        model.commit()
        assert call("commit", None)[0] == 0
    # without a standing step: no rows
    error, positions, masks = trees.call()
    assert error == 0 and (positions == -1).all() and (masks == 0).all()


@pytest.mark.gpu
def test_bad_parents_and_trees_too_large_are_reported(pcl, torch, ctx):
    shape = (3, 20, 16, 50, 200)
    trees = Trees(pcl, torch, ctx, shape, 1)
    model = ShareModel(*shape)
    call = tp.device_call(ctx, trees.batch)
    ctx.page_reset(trees.batch.desc)
    assert model.step([9, 4, 0]) and call("step", [9, 4, 0])[0] == 0
    model.commit(), call("commit", None)
    assert model.step([6, 0, 70]) and call("step", [6, 0, 70])[0] == 0
    parents = [[-1, 0, 1, 1, 3, 4], [], [i - 1 for i in range(70)]]
    trees.put(parents)
    error, positions, masks = trees.call()
    assert error == BAD_PAGES  # 70 tokens in 64 bits: the held ones alone
    want = expected(model, [parents[0], [], []], 200, 1)
    assert np.array_equal(positions[:6], want[0][:6]) and np.array_equal(masks[:6], want[1][:6])
    assert positions[6:76].tolist() == list(range(70)) and (masks[6:] == 0).all()
    assert (positions[76:] == -1).all()
    assert model.step([6, 0, 4]) and call("step", [6, 0, 4])[0] == 0
    for bad in (3, 4, 5, -2, 1 << 30, -(1 << 31)):
        trees.put([[-1, 0, 1, bad, 3, 4], [], [-1, 0, 0, 2]])
        error, positions, masks = trees.call()
        assert error == BAD_PAGES
        # its own token and no other, as one that follows the held ones
        want = expected(model, [[-1, 0, 1, -1, 3, 4], [], [-1, 0, 0, 2]], 200, 1)
        assert np.array_equal(positions, want[0]) and np.array_equal(masks, want[1])


def accept_call(ctx, torch, batch, paths, counts, depth):
    dev = {"device": "cuda:0"}
    p = torch.full((len(counts), depth), 1 << 20, dtype=torch.int32, **dev)
    for b, x in enumerate(paths):
        p[b, :len(x)] = torch.tensor(x, dtype=torch.int32)
    c = torch.tensor(counts, dtype=torch.int32, **dev)
    moves = [torch.full_like(p, 99) for _ in range(2)]
    ctx.page_accept(batch.desc, p.data_ptr(), c.data_ptr(), depth,
                    *[x.data_ptr() for x in moves])
    error = ctx.sync()
    return error, moves


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 9, 7, 30, 90), (6, 40, 16, 200, 700),
                                   (130, 9, 5, 900, 1300)], ids=str)
def test_accepted_branches_follow_the_model(pcl, torch, ctx, shape):
    rng = np.random.default_rng(shape[0])
    batch = DeviceBatch(pcl, torch, *shape)
    model = ShareModel(*shape)
    call = tp.device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    room = shape[1] * shape[2]
    for turn in range(4):
        counts = [int(min(rng.integers(0, 9), room - n)) for n in model.lengths]
        if turn == 2:
            counts[0] = min(70, room - model.lengths[0])  # more than a wave's lanes
        assert model.step(counts) and call("step", counts)[0] == 0
        paths = [sorted(rng.permutation(n)[:int(rng.integers(0, n + 1))].tolist())
                 for n in counts]
        depth = max([len(x) for x in paths] + [1]) + turn
        lens = [len(x) for x in paths]
        error, (source, target) = accept_call(ctx, torch, batch, paths, lens, depth)
        assert error == 0
        want = np.full((2, shape[0], depth), -1)
        for b, path in enumerate(paths):
            held = model.lengths[b]
            for k, i in enumerate(path):
                if i != k:
                    for w, x in zip(want, (held + i, held + k)):
                        w[b, k] = model.table[b][x // shape[2]] * shape[2] + x % shape[2]
        assert np.array_equal(source.cpu().numpy(), want[0])
        assert np.array_equal(target.cpu().numpy(), want[1])
        model.check(batch.state())
        assert model.commit(lens) and call("commit", lens)[0] == 0
        model.check(batch.state())
    # no standing step: nothing moves
    error, moves = accept_call(ctx, torch, batch, [[]] * shape[0], [0] * shape[0], 3)
    assert error == 0 and all(bool((x == -1).all()) for x in moves)


@pytest.mark.gpu
def test_branches_that_are_none_are_not_committed(pcl, torch, ctx):
    shape = (2, 30, 8, 60, 300)
    batch = DeviceBatch(pcl, torch, *shape)
    call = tp.device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    assert call("step", [5, 3])[0] == 0 and call("commit", None)[0] == 0
    for paths, counts, depth in (
            ([[1, 1], [0]], [2, 1], 2), ([[2, 1], [0]], [2, 1], 2), ([[0, 90], [0]], [2, 1], 2),
            ([[-1], [0]], [1, 1], 2), ([[0, 1, 2], [0]], [-1, 1], 3),
            ([[0, 1], [0, 1, 2]], [2, 3], 2),  # more than depth
            ([[0], [0, 1, 2, 3, 4]], [1, 5], 5),  # more than the new tokens
            ([list(range(64)) + [80, 70], [0]], [66, 1], 70)):
        assert call("step", [90, 4])[0] == 0
        depth_counts = [min(len(x), depth) for x in paths]
        error, (source, target) = accept_call(
            ctx, torch, batch, [x[:n] for x, n in zip(paths, depth_counts)], counts, depth)
        assert error == BAD_PAGES, paths
        bad = 0 if counts[0] != 1 and len(paths[1]) < 3 or paths[0] == [-1] else 1
        assert bool((source[bad] == -1).all()) and bool((target[bad] == -1).all())
        state = batch.state()
        assert state["counters"][3] == 0
        before = [state[n].copy() for n in ("lengths", "counters", "free_pages")]
        assert call("commit", [1, 1])[0] == 0
        assert all(np.array_equal(x, y) for x, y in zip(before, [
            batch.state()[n] for n in ("lengths", "counters", "free_pages")]))
    # a page outside the pools under a branch
    assert call("step", [90, 4])[0] == 0
    batch.a["table"][5] = 60
    error, moves = accept_call(ctx, torch, batch, [[0, 40], [0]], [2, 1], 2)
    assert error == BAD_PAGES and bool((moves[0][0] == -1).all())


# ---- shared pages on the device ----------------------------------------------------

def fork_call(ctx, torch, batch, sources):
    n = len(sources)
    out = [torch.full((n,), 99, dtype=torch.int32, device="cuda:0") for _ in range(3)]
    ctx.page_fork(batch.desc, batch.put(sources), *[x.data_ptr() for x in out])
    return ctx.sync(), [x.tolist() for x in out]


def release_call(ctx, batch, finished):
    ctx.page_release_shared(batch.desc, batch.put(finished))
    return ctx.sync(), batch.state()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 9, 7, 20, 130), (5, 40, 1, 90, 64), (37, 6, 16, 120, 700),
                                   (300, 3, 8, 500, 900), (2048, 2, 4, 2600, 2500),
                                   # more table entries, and pages, than one workgroup takes
                                   (2048, 9, 4, 2600, 2500), (40, 450, 1, 3001, 900),
                                   (6, 8, 16, 131073 + 40, 300)],
                         ids=lambda s: "x".join(map(str, s)))
def test_shared_bookkeeping_follows_the_model(pcl, torch, ctx, shape):
    rng = np.random.default_rng(sum(shape))
    batch = DeviceBatch(pcl, torch, *shape)
    model = ShareModel(*shape)
    call = tp.device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    forks = 0
    for turn in range(24):
        room = [shape[1] * shape[2] - n for n in model.lengths]
        counts = [int(min(r, c)) for r, c in zip(room, rng.choice([0, 0, 1, 2, 9], shape[0]))]
        budget = min(shape[4], len(model.free) * shape[2] // 2)
        for b in range(shape[0]):
            counts[b] = max(0, min(counts[b], budget))
            budget -= counts[b]
        ok = model.step(counts)
        assert call("step", counts)[0] == (0 if ok else BAD_PAGES)
        if ok and rng.random() < 0.8:
            model.commit()
            assert call("commit", None)[0] == 0
        model.check(batch.state())
        # free slots begin as copies of random requests; now and then one that may not
        sources = [-1] * shape[0]
        free = [b for b, n in enumerate(model.lengths) if n == 0]
        held = [b for b, n in enumerate(model.lengths) if n > 0]
        if held:
            for b in free:
                if rng.random() < 0.6:
                    sources[b] = int(rng.choice(held))
            if rng.random() < 0.2:
                sources[int(rng.integers(shape[0]))] = int(rng.choice([held[0], shape[0]]))
        want = model.fork(sources)
        error, got = fork_call(ctx, torch, batch, sources)
        assert error == (0 if want else BAD_PAGES)
        assert got == (want or [[-1] * shape[0]] * 2 + [[0] * shape[0]])
        model.check(batch.state())
        forks += want is not None and any(s >= 0 for s in sources)
        if want and rng.random() < 0.8:
            model.commit()
            assert call("commit", None)[0] == 0
            model.check(batch.state())
        finished = [int(f) for f in rng.random(shape[0]) < rng.choice([0.1, 0.5])]
        model.release_shared(finished)
        error, state = release_call(ctx, batch, finished)
        assert error == 0
        for name, x in (("lengths", model.lengths), ("free_pages", model.free),
                        ("counters", [len(model.free)])):
            assert state[name][:len(x)].tolist() == x
        assert state["counters"][3] == 0
        # every page is free, or held, and never both
        held = {p for b in range(shape[0]) for p in model.pages_of(b)}
        assert len(set(model.free)) == len(model.free)
        assert not held & set(model.free) and len(held) + len(model.free) == shape[3]
    assert forks > 3
    everyone = [1] * shape[0]
    model.release_shared(everyone)
    error, state = release_call(ctx, batch, everyone)
    assert error == 0 and state["free_pages"].tolist() == model.free
    assert len(model.free) == shape[3]


@pytest.mark.gpu
def test_forks_that_do_not_stand(pcl, torch, ctx):
    shape = (5, 8, 8, 12, 100)
    batch = DeviceBatch(pcl, torch, *shape)
    model = ShareModel(*shape)
    call = tp.device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    assert model.step([20, 17, 0, 0, 0]) and call("step", [20, 17, 0, 0, 0])[0] == 0
    model.commit(), call("commit", None)
    good = {n: x.clone() for n, x in batch.a.items()}

    def held():
        return [batch.state()[n] for n in ("lengths", "counters", "free_pages")]

    # a fork keeps what its source holds: a commit of a part is refused
    model.fork([-1, -1, 0, 0, 1])
    assert fork_call(ctx, torch, batch, [-1, -1, 0, 0, 1])[0] == 0
    before = held()
    for kept in ([0, 0, 20, 20, 17], [0] * 5, [0, 0, 8, 0, 0]):
        assert call("commit", kept)[0] == BAD_PAGES
        assert all(np.array_equal(x, y) for x, y in zip(before, held()))
    # (it still stands)
    model.commit()
    assert call("commit", None)[0] == 0
    model.check(batch.state())
    # the plain release refuses what they share, the other one gives back the rest
    assert call("release", [1, 0, 0, 0, 0])[0] == BAD_PAGES
    model.release_shared([1, 0, 0, 1, 0])
    error, state = release_call(ctx, batch, [1, 0, 0, 1, 0])
    assert error == 0 and state["free_pages"][:len(model.free)].tolist() == model.free
    for n, x in good.items():
        batch.a[n].copy_(x)
    # too few free pages
    batch.a["counters"][0] = 2
    error, got = fork_call(ctx, torch, batch, [-1, -1, 0, 0, 1])
    assert error == BAD_PAGES and got == [[-1] * 5, [-1] * 5, [0] * 5]
    assert torch.equal(batch.a["table"], good["table"])
    assert batch.a["counters"].tolist() == [2, 0, 0, 0]
    batch.a["counters"].copy_(good["counters"])
    # lengths outside the table
    for b, bad in ((0, 65), (3, -1), (4, 1 << 30)):
        batch.a["lengths"][b] = bad
        assert fork_call(ctx, torch, batch, [-1, -1, 0, -1, -1])[0] == BAD_PAGES
        assert torch.equal(batch.a["table"], good["table"])
        batch.a["lengths"].copy_(good["lengths"])
    # pages outside the pools: under the last tokens, and on the free list
    top = int(good["counters"][0]) - 1
    for name, at in (("table", 2), ("free_pages", top)):
        for bad in (12, -1, 1 << 30, -(1 << 31)):
            batch.a[name][at] = bad
            error, got = fork_call(ctx, torch, batch, [-1, -1, 0, -1, -1])
            assert error == BAD_PAGES and got == [[-1] * 5, [-1] * 5, [0] * 5]
            before = held()
            assert before[1][3] == 0 and call("commit", None)[0] == 0
            assert all(np.array_equal(x, y) for x, y in zip(before, held()))
            for n, x in good.items():
                batch.a[n].copy_(x)
    # a fork writes no rows, and drops a step's
    assert call("step", [1, 1, 1, 0, 0])[0] == 0
    model = None
    assert fork_call(ctx, torch, batch, [-1, -1, 0, -1, -1])[0] == 0
    state = batch.state()
    for n in ("slots", "positions", "row_request", "newest"):
        assert (state[n] == -1).all()
    # a fork of a request without tokens holds none
    error, got = fork_call(ctx, torch, batch, [-1, -1, 3, -1, -1])
    assert error == 0 and got == [[-1] * 5, [-1] * 5, [0] * 5]
    assert call("commit", None)[0] == 0 and batch.state()["lengths"].tolist() == [20, 17, 0, 0, 0]


@pytest.mark.gpu
def test_shared_releases_that_are_refused(pcl, torch, ctx):
    shape = (4, 6, 8, 24, 100)
    batch = DeviceBatch(pcl, torch, *shape)
    call = tp.device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    assert call("step", [20, 30, 9, 5])[0] == 0 and call("commit", None)[0] == 0
    assert call("step", [1, 1, 1, 1])[0] == 0
    good = {n: x.clone() for n, x in batch.a.items()}

    def refused(finished):
        before = batch.state()
        error, after = release_call(ctx, batch, finished)
        assert error == BAD_PAGES
        for n in STATE:
            assert np.array_equal(before[n], after[n]), n
        for n, x in good.items():
            batch.a[n].copy_(x)

    for bad in (24, -1, 1 << 30, -(1 << 31)):
        batch.a["table"][1] = bad  # among the finished request's pages
        refused([1, 0, 0, 0])
        batch.a["free_pages"][2] = bad
        refused([1, 0, 0, 0])
    batch.a["table"][1] = batch.a["free_pages"][0]  # free already
    refused([1, 1, 0, 0])
    for bad in (-1, 49, 1 << 30):
        batch.a["lengths"][2] = bad
        refused([1, 0, 0, 0])
    for bad in (-1, 25):
        batch.a["counters"][0] = bad
        refused([1, 0, 0, 0])
    # a page outside the pools that stays is not looked at
    batch.a["table"][1] = 24
    error, state = release_call(ctx, batch, [0, 0, 1, 1])
    assert error == 0 and state["lengths"].tolist() == [20, 30, 0, 0]
    # a page twice in one table goes back once
    for n, x in good.items():
        batch.a[n].copy_(x)
    batch.a["table"][1] = batch.a["table"][0]
    n = int(good["counters"][0])
    error, state = release_call(ctx, batch, [1, 0, 0, 0])
    assert error == 0 and state["free_pages"][n:n + 2].tolist() == [2, 0]
    assert state["counters"][0] == n + 2
    # nobody
    error, state = release_call(ctx, batch, [0, 0, 0, 0])
    assert error == 0 and state["counters"][0] == n + 2


# ---- copies -------------------------------------------------------------------------

def copy_model(pool, lists):
    """Rows of a pool [slots][...] after the lists of (from, to, rows)."""
    out = pool.clone()
    for entries in lists:
        for a, b, n in entries:
            if a >= 0 and b >= 0 and n > 0:
                out[b:b + n] = out[a:a + n].clone()
    return out


def layers_of(pcl, torch, pages, page, kinds, seed):
    g = torch.Generator(device="cuda:0")
    g.manual_seed(seed)
    out = []
    for kvheads, dim, dtype in kinds:
        pools = Pools(pcl, torch, pages, page, kvheads, dim, dtype)
        for x in (pools.k, pools.v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda:0"))
        out.append(pools)
    return out


KINDS = [(2, 16, "f32"), (1, 48, "bf16"), (8, 256, "bf16"), (3, 512, "f32"), (40, 64, "f32"),
         (1, 16, "bf16")]


def check_copies(pcl, torch, ctx, layers, lists, rows):
    flat = [[x.view(-1, *x.shape[2:]).clone() for x in (p.k, p.v)] for p in layers]
    dev = {"dtype": torch.int32, "device": "cuda:0"}
    entries = len(lists[0])
    source, target, count = (torch.tensor([[e[i] for e in x] for x in lists], **dev)
                             for i in range(3))
    ctx.paged_copy([p.desc for p in layers], source.data_ptr(), target.data_ptr(), len(lists),
                   entries, count.data_ptr() if rows else None)
    assert ctx.sync() == 0
    for p, before in zip(layers, flat):
        for x, old in zip((p.k, p.v), before):
            assert torch.equal(x.view(-1, *x.shape[2:]), copy_model(old, lists))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 7, 64])
def test_runs_are_copied(pcl, torch, ctx, page):
    rng = np.random.default_rng(page)
    pages = 40
    layers = layers_of(pcl, torch, pages, page, KINDS, page)
    order = rng.permutation(pages)
    lists = []
    for i in range(18):
        n = int(rng.integers(0, page + 1)) if i else page
        a, b = (int(order[j]) * page + int(rng.integers(0, page - n + 1))
                for j in (2 * i, 2 * i + 1))
        lists.append([(-1 if i == 5 else a, -1 if i == 9 else b, -3 if i == 11 else n)])
    check_copies(pcl, torch, ctx, layers, lists, True)
    # several pages at once, up to the pools' last row; and one row each
    lists = [[(0, pages * page - 9 * page, 9 * page)], [(9 * page, 20 * page, 5 * page)]]
    check_copies(pcl, torch, ctx, layers, lists, True)
    lists = [[(int(a) * page, int(b) * page, 1)] for a, b in zip(order[:15], order[15:30])]
    check_copies(pcl, torch, ctx, layers, lists, False)


@pytest.mark.gpu
@pytest.mark.parametrize("entries", [2, 8, 9, 40])
def test_lists_are_copied_in_order(pcl, torch, ctx, entries):
    rng = np.random.default_rng(entries)
    page = 16
    each = -(-(3 * entries + 5) // page)
    layers = layers_of(pcl, torch, 6 * each + 2, page, KINDS, entries)
    order = rng.permutation(6 * each).reshape(6, each)
    lists = []
    for b in range(6):
        slot = (order[b][:, None] * page + np.arange(page)).reshape(-1)
        # branches that begin at their place, one behind it, and at random
        path = sorted(rng.permutation(3 * entries)[:entries].tolist())
        path = [list(range(entries)), list(range(1, entries + 1)), path][b % 3]
        lists.append([(int(slot[i]) if i != k and (b, k) != (4, 1) else -1, int(slot[k]), 1)
                      for k, i in enumerate(path)])
    check_copies(pcl, torch, ctx, layers, lists, False)


@pytest.mark.gpu
def test_more_layers_than_one_launch_copies(pcl, torch, ctx):
    layers = layers_of(pcl, torch, 4, 3, [(1, 16 * (1 + i % 3), "f32") for i in range(131)], 3)
    check_copies(pcl, torch, ctx, layers, [[(0, 6, 3)], [(4, 9, 1)]], True)
    check_copies(pcl, torch, ctx, layers, [[(1, 0, 1), (2, 1, 1)], [(5, 4, 1), (11, 5, 1)]], False)


@pytest.mark.gpu
def test_copies_past_the_pools_are_reported(pcl, torch, ctx):
    page, pages = 5, 3
    layers = layers_of(pcl, torch, pages, page, [(2, 64, "f32"), (1, 32, "bf16")], 5)
    old = [x.clone() for p in layers for x in (p.k, p.v)]
    dev = {"dtype": torch.int32, "device": "cuda:0"}
    big = (1 << 31) - 1
    for a, b, n in ((0, 15, 1), (15, 0, 1), (0, 11, 5), (11, 0, 5), (0, 5, big), (big, 0, 1),
                    (0, big, 2), (0, 1 << 30, 1)):
        words = [torch.tensor(x, **dev) for x in ([a, 7], [b, 8], [n, 1])]
        for x, y in zip([x for p in layers for x in (p.k, p.v)], old):
            x.copy_(y)
        ctx.paged_copy([p.desc for p in layers], words[0].data_ptr(), words[1].data_ptr(), 2, 1,
                       words[2].data_ptr())
        assert ctx.sync() == BAD_PAGES
        want = [copy_model(y.view(15, *y.shape[2:]), [[(7, 8, 1)]]) for y in old]
        for x, y in zip([x for p in layers for x in (p.k, p.v)], want):
            assert torch.equal(x.view(y.shape), y)
        if n == 1:  # in a list too
            words = [torch.tensor(x, **dev) for x in ([[a, 7]], [[b, 8]])]
            for x, y in zip([x for p in layers for x in (p.k, p.v)], old):
                x.copy_(y)
            ctx.paged_copy([p.desc for p in layers], words[0].data_ptr(), words[1].data_ptr(), 1,
                           2)
            assert ctx.sync() == BAD_PAGES
            for x, y in zip([x for p in layers for x in (p.k, p.v)], want):
                assert torch.equal(x.view(y.shape), y)


@pytest.mark.gpu
def test_copies_past_32_bit_offsets(pcl, torch, ctx):
    kvheads, dim, page = 8, 256, 64
    pages = (1 << 31) // (page * kvheads * dim) + 40
    k = torch.empty((pages, page, kvheads, dim), device="cuda:0", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    pools = pcl.page_pools(k=k.data_ptr(), v=v.data_ptr(), type=pcl.CACHE_BF16, pages=pages,
                           page_tokens=page, kvheads=kvheads, dim=dim)
    for x in (k, v):
        x[pages - 2].normal_()
        x[3].zero_()
        x[pages - 1].zero_()
    dev = {"dtype": torch.int32, "device": "cuda:0"}
    words = [torch.tensor(x, **dev) for x in ([(pages - 2) * page + 3, (pages - 2) * page],
                                              [3 * page, (pages - 1) * page], [50, page])]
    ctx.paged_copy([pools], words[0].data_ptr(), words[1].data_ptr(), 2, 1, words[2].data_ptr())
    assert ctx.sync() == 0
    for x in (k, v):
        assert torch.equal(x[3, :50], x[pages - 2, 3:53]) and bool((x[3, 50:] == 0).all())
        assert torch.equal(x[pages - 1], x[pages - 2])


# ---- attention ----------------------------------------------------------------------

class TreeCache(Cache):
    """Requests that hold tokens and have new ones: rows in the requests' order, or
    anywhere (`first`). masks: None for a chain, else per request [n][n] booleans."""

    def __init__(self, pcl, torch, heads, held, counts, page, dtype, seed, masks=None,
                 positions=None, first=None, rows=None, scale=1.0):
        super().__init__(pcl, torch, heads, [a + n for a, n in zip(held, counts)], page, dtype,
                         seed, scale)
        self.held, self.counts, self.masks = list(held), list(counts), masks
        starts = np.concatenate(([0], np.cumsum(counts)))
        self.first = list(starts[:-1]) if first is None else first
        self.rows = int(starts[-1]) + 3 if rows is None else rows
        dev = {"dtype": torch.int32, "device": "cuda:0"}
        self.dheld = torch.tensor(self.held, **dev)
        self.newest = torch.tensor([f + n - 1 if n else -1
                                    for f, n in zip(self.first, counts)], **dev)
        self.positions = positions or [[a + i for i in range(n)] for a, n in zip(held, counts)]
        self.words = max(1, -(-max(list(counts) + [1]) // 64))
        if masks is not None:
            m = np.zeros((self.rows, self.words), np.int64)
            p = np.full(self.rows, -1)
            for b, n in enumerate(counts):
                for i in range(n):
                    m[self.first[b] + i] = words_of(np.flatnonzero(masks[b][i]), self.words)
                    p[self.first[b] + i] = self.positions[b][i]
            self.dmasks = torch.from_numpy(m).to("cuda:0")
            self.dpositions = torch.tensor(p, **dev)

    def sees(self, b, window=0):
        """Which keys each new token of request b attends, [n][keys]."""
        a, n = self.held[b], self.counts[b]
        s = np.ones((n, a + n), bool)
        s[:, a:] = np.tril(np.ones((n, n), bool)) if self.masks is None else self.masks[b]
        at = np.concatenate((np.arange(a), self.positions[b]))
        if window:
            s &= np.array(self.positions[b])[:, None] - at[None, :] < window
        return s

    def tree_desc(self, ctx, q, out, window=0, softcap=0.0, max_length=None, max_new=None, **kw):
        qheads, _, dim = self.heads
        tree = {}
        if self.masks is not None:
            tree = dict(masks=self.dmasks.data_ptr(), mask_words=self.words,
                        positions=self.dpositions.data_ptr())
        fields = dict(
            pools=self.pools.desc, q=q.data_ptr(), q_stride=q.stride(0), q_rows=q.shape[0],
            qheads=qheads, table=self.table.data_ptr(), table_stride=self.stride,
            lengths=self.dheld.data_ptr(), step_lengths=self.dlengths.data_ptr(),
            newest=self.newest.data_ptr(), requests=len(self.held),
            max_length=max_length or self.stride * self.page,
            max_new=max_new or max(self.counts + [1]), window=window, q_scale=scale_of(dim),
            softcap=softcap, out=out.data_ptr(), o_stride=out.stride(0), **tree)
        fields.update(kw)
        return ctx.paged_tree_desc(**fields)

    def tree_attend(self, ctx, q, out=None, **kw):
        torch = self.torch
        out = torch.full_like(q, 9.5) if out is None else out
        torch.cuda.synchronize()
        ctx.paged_tree_attention(self.tree_desc(ctx, q, out, **kw))
        torch.cuda.synchronize()
        return out

    def queries(self, seed=1, scale=1.0):
        g = self.torch.Generator(device="cuda:0")
        g.manual_seed(seed)
        return scale * self.torch.randn((self.rows, self.heads[0] * self.heads[2]), generator=g,
                                        device="cuda:0")

    def contiguous_rows(self, ctx, q, b, window=0, softcap=0.0):
        """Request b's new tokens through pcl_attention_launch: causal, or with the
        keys that they see as bytes."""
        torch = self.torch
        qheads, kvheads, dim = self.heads
        n, a = self.counts[b], self.held[b]
        q = q[self.first[b]:self.first[b] + n, :qheads * dim].contiguous()
        out = torch.empty_like(q)
        k, v = self.k[b].contiguous(), self.v[b].contiguous()
        kw = dict(causal=1, window=window, first_query=a)
        if self.masks is not None:
            seen = self.sees(b, window)
            mask = torch.from_numpy(seen.astype(np.uint8)).to("cuda:0")
            kw = dict(mask=mask.data_ptr(), mask_stride=a + n)
        torch.cuda.synchronize()
        ctx.launch(ctx.desc(
            q=q.data_ptr(), q_stride=qheads * dim, nq=n, k0=k.data_ptr(), v0=v.data_ptr(),
            n0=a + n, qheads=qheads, kvheads=kvheads, dim=dim, kh_first=0, kh_end=kvheads,
            q_scale=scale_of(dim), softcap=softcap, out=out.data_ptr(), o_stride=qheads * dim,
            **kw))
        torch.cuda.synchronize()
        return out

    def exact_rows(self, q, b, window=0, softcap=0.0):
        """Request b's new tokens in 64 bits and a bound of the kernels' error for
        each value: exact_and_bound of test_paged.py over the keys that each token
        sees (its derivation holds for any set of keys)."""
        torch = self.torch
        qheads, kvheads, dim = self.heads
        n, keys = self.counts[b], self.lengths[b]
        seen = torch.from_numpy(self.sees(b, window)).to("cuda:0")[None, :, None, :]
        x = (q[self.first[b]:self.first[b] + n, :qheads * dim] * np.float32(scale_of(dim)))
        x = x.double().view(n, kvheads, -1, dim).transpose(0, 1).contiguous()
        k, v = self.k[b].double(), self.v[b].double()
        kt = k.permute(1, 2, 0).contiguous()[:, None]
        vt = v.permute(1, 0, 2).contiguous()[:, None]
        s, size = torch.matmul(x, kt), torch.matmul(x.abs(), kt.abs())
        capped = softcap * torch.tanh(s / softcap) if softcap else s
        low = torch.where(seen, capped, float("inf")).amin(-1, keepdim=True)
        capped = torch.where(seen, capped, -float("inf"))
        top = capped.amax(-1, keepdim=True)
        w = torch.softmax(capped, -1)
        exact = torch.matmul(w, vt)
        biggest = torch.maximum(top.abs(), low.abs())
        spans = keys // (16 * 256) + 1
        e = 1.01 * dim * torch.where(seen, size, 0.0).amax(-1, keepdim=True) + \
            (20 * biggest if softcap else 0) + 3 * (top - low) + \
            2 * (1 + 8 + 17 + spans + 1) + 256 + 8 + 16 + spans + 2
        u = 2.0 ** -24
        bound = 2.02 * e * u * torch.matmul(w, vt.abs()) + 4 * u * exact.abs()
        return [y.transpose(0, 1).reshape(n, qheads * dim) for y in (exact, bound)]

    def check(self, ctx, q, out, requests=None, window=0, softcap=0.0, exact=True):
        qd = self.heads[0] * self.heads[2]
        for b in range(len(self.held)) if requests is None else requests:
            n = self.counts[b]
            if n == 0:
                continue
            got = out[self.first[b]:self.first[b] + n, :qd]
            want = self.contiguous_rows(ctx, q, b, window, softcap)
            # adding 0 makes a negative zero positive
            assert np.array_equal(bits(got + 0.0), bits(want + 0.0)), (b, self.held[b], n)
            if exact:
                value, bound = self.exact_rows(q, b, window, softcap)
                assert bool(((got.double() - value).abs() <= bound).all()), (b, self.held[b], n)


def random_trees(rng, held, counts):
    """(masks, positions) of random trees."""
    masks, positions = [], []
    for a, n in zip(held, counts):
        depth, branch = tree_of(random_parents(rng, n))
        m = np.zeros((n, n), bool)
        for i, x in enumerate(branch):
            m[i, list(x)] = True
        masks.append(m)
        positions.append([a + d for d in depth])
    return masks, positions


HEADS = [(16, 8, 256), (16, 2, 512), (32, 8, 128), (16, 4, 64), (10, 2, 80), (3, 3, 16),
         (20, 1, 48), (2, 1, 272), (33, 1, 128)]
# held and new tokens: nothing held, one token, around tiles, pages and chunks, new
# tokens across a chunk's end, several chunks, more than one span
HELD = [0, 0, 1, 15, 31, 33, 200, 255, 256, 250, 511, 1000, 4090, 5000, 77]
COUNTS = [1, 9, 1, 3, 2, 5, 70, 1, 7, 13, 4, 1, 12, 3, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_attention_has_the_contiguous_bits(pcl, torch, ctx, dtype, heads, window, tree):
    page = {256: 16, 512: 7, 128: 48, 64: 300}.get(heads[2], 5)
    rng = np.random.default_rng(heads[2] + window)
    masks = positions = None
    if tree:
        masks, positions = random_trees(rng, HELD, COUNTS)
    cache = TreeCache(pcl, torch, heads, HELD, COUNTS, page, dtype, heads[2] + window, masks,
                      positions)
    q = cache.queries()
    out = cache.tree_attend(ctx, q, window=window)
    assert ctx.sync() == 0
    cache.check(ctx, q, out, window=window)
    assert bool((out[cache.rows - 3:] == 9.5).all())
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(4, 4, 64), (16, 2, 64), (12, 1, 64), (8, 4, 128), (5, 1, 128),
                                   (16, 8, 256), (14, 2, 256), (4, 2, 512), (16, 2, 512),
                                   (2, 1, 496)], ids=lambda h: "x".join(map(str, h)))
def test_launches_of_few_items(pcl, torch, ctx, dtype, heads):
    rng = np.random.default_rng(heads[2])
    for held, counts in (([0], [1]), ([100], [6]), ([257, 40], [2, 1]), ([64, 2, 700], [1, 4, 2]),
                         ([30, 500], [40, 17])):
        masks, positions = random_trees(rng, held, counts)
        cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, sum(held), masks, positions)
        q = cache.queries()
        out = cache.tree_attend(ctx, q, max_length=max(cache.lengths))
        loose = cache.tree_attend(ctx, q, max_new=300)
        assert ctx.sync() == 0
        cache.check(ctx, q, out)
        assert np.array_equal(bits(loose), bits(out))
        assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype", [((16, 8, 256), "bf16"), ((16, 2, 512), "f32"),
                                         ((4, 4, 64), "bf16"), ((32, 8, 128), "f32")], ids=str)
@pytest.mark.parametrize("window", [0, 700])
def test_parts_of_prompts(pcl, torch, ctx, heads, dtype, window):
    # many new tokens behind held ones: several units, chunks before and behind
    held, counts = [900, 0, 300, 2000, 5], [300, 600, 1, 129, 64]
    cache = TreeCache(pcl, torch, heads, held, counts, 32, dtype, 5)
    q = cache.queries()
    out = cache.tree_attend(ctx, q, window=window)
    assert ctx.sync() == 0
    cache.check(ctx, q, out, window=window)
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(16, 8, 256), (16, 2, 512)], ids=["d256", "d512"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_requests(pcl, torch, ctx, heads, dtype):
    # several spans; one request alone and among others has the same bits
    held, counts = [20000, 3, 40001, 9000], [5, 2, 33, 8]
    masks, positions = random_trees(np.random.default_rng(3), held, counts)
    cache = TreeCache(pcl, torch, heads, held, counts, 64, dtype, 11, masks, positions)
    q = cache.queries()
    out = cache.tree_attend(ctx, q)
    cache.check(ctx, q, out)
    windowed = cache.tree_attend(ctx, q, window=6000)
    cache.check(ctx, q, windowed, window=6000, exact=False)
    newest = cache.newest.clone()
    for b in range(4):
        cache.newest.fill_(-1)
        cache.newest[b] = newest[b]
        alone = cache.tree_attend(ctx, q)
        mine = slice(cache.first[b], cache.first[b] + counts[b])
        assert np.array_equal(bits(alone[mine]), bits(out[mine]))
        alone[mine] = 9.5
        assert bool((alone == 9.5).all())
    assert ctx.sync() == 0


@pytest.mark.gpu
def test_windows_inside_the_trees(pcl, torch, ctx):
    # windows shorter than a branch: ancestors fall out of them, and held tokens too
    for heads, dtype in (((16, 8, 256), "f32"), ((5, 1, 64), "bf16"), ((4, 4, 128), "f32")):
        held, counts = [0, 3, 250, 600, 7], [40, 20, 30, 64, 1]
        masks, positions = [], []
        for a, n in zip(held, counts):  # two long branches
            depth, branch = tree_of([-1, -1] + list(range(n - 2)) if n > 1 else [-1])
            m = np.zeros((n, n), bool)
            for i, x in enumerate(branch):
                m[i, list(x)] = True
            masks.append(m)
            positions.append([a + d for d in depth])
        cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, 4, masks, positions)
        q = cache.queries()
        for window in (1, 2, 5, 17, 300):
            out = cache.tree_attend(ctx, q, window=window)
            assert ctx.sync() == 0
            cache.check(ctx, q, out, window=window)
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1 << 31, (1 << 63) - 1])
def test_a_window_without_a_limit(pcl, torch, ctx, window):
    held, counts = [700, 3], [5, 9]
    masks, positions = random_trees(np.random.default_rng(1), held, counts)
    for tree in (None, masks):
        cache = TreeCache(pcl, torch, (4, 2, 64), held, counts, 16, "f32", 4, tree,
                          positions if tree else None)
        q = cache.queries()
        assert np.array_equal(bits(cache.tree_attend(ctx, q, window=window)),
                              bits(cache.tree_attend(ctx, q)))
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.75, 50.0])
def test_softcap(pcl, torch, ctx, softcap):
    for heads, dtype in (((16, 8, 256), "f32"), ((32, 8, 128), "bf16"), ((10, 2, 80), "f32")):
        held, counts = [0, 300, 700], [3, 20, 7]
        masks, positions = random_trees(np.random.default_rng(2), held, counts)
        cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, 3, masks, positions)
        q = cache.queries(scale=6.0)
        out = cache.tree_attend(ctx, q, softcap=softcap)
        assert ctx.sync() == 0
        cache.check(ctx, q, out, softcap=softcap)
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 1, 64), (3, 3, 128), (16, 2, 512)],
                         ids=lambda h: "x".join(map(str, h)))
def test_any_masks(pcl, torch, ctx, heads):
    # bits that are no tree's: tokens without themselves, that see later ones, that
    # see nothing; keys that nobody sees hold NaNs and infinities
    rng = np.random.default_rng(heads[2])
    held, counts = [0, 40, 0, 254, 600], [30, 12, 70, 9, 130]
    masks = [rng.random((n, n)) < 0.3 for n in counts]
    for m in masks:
        m[:, [2, -1]] = False
        m[4] = False
    masks[0][:, 8:16] = False
    cache = TreeCache(pcl, torch, heads, held, counts, 16, "f32", 4, masks)
    for b, (a, n) in enumerate(zip(held, counts)):
        for j in np.flatnonzero(~masks[b].any(0)):
            at = a + int(j)
            slot = int(cache.table[b, at // 16]) * 16 + at % 16
            for x, keep, bad in ((cache.pools.k, cache.k, float("nan")),
                                 (cache.pools.v, cache.v, float("inf") if j % 2 else float("nan"))):
                x.view(-1, *x.shape[2:])[slot] = bad
                keep[b][at] = 0.0  # (the contiguous rows: any value)
    q = cache.queries()
    out = cache.tree_attend(ctx, q)
    assert ctx.sync() == 0
    for b, (a, n) in enumerate(zip(held, counts)):
        mine = out[cache.first[b]:cache.first[b] + n]
        some = torch.from_numpy(cache.sees(b).any(1)).to("cuda:0")
        assert bool((mine[~some] == 9.5).all()) and bool((~some).any()) == (a == 0)
        want = cache.contiguous_rows(ctx, q, b)
        assert np.array_equal(bits(mine[some] + 0.0), bits(want[some] + 0.0)), b
        value, bound = cache.exact_rows(q, b)
        assert bool(((mine.double() - value).abs() <= bound)[some].all())
    ctx.sync()  # (the contiguous launch reports the rows without keys)


@pytest.mark.gpu
def test_values_that_nobody_sees_at_the_ends(pcl, torch, ctx):
    # whole tiles, and a whole chunk, of new tokens that no token of the batch sees
    heads = (4, 2, 64)
    held, counts = [250, 3], [300, 400]
    masks = [np.eye(n, dtype=bool) for n in counts]
    for m in masks:
        m[6:280] = False
        m[:, 6:280] = False
        m[6:280, 0] = True
    cache = TreeCache(pcl, torch, heads, held, counts, 16, "bf16", 4, masks)
    for b, (a, n) in enumerate(zip(held, counts)):
        for at in range(a + 6, a + 280):
            slot = int(cache.table[b, at // 16]) * 16 + at % 16
            for x, keep in ((cache.pools.k, cache.k), (cache.pools.v, cache.v)):
                x.view(-1, *x.shape[2:])[slot] = float("nan")
                keep[b][at] = 0.0
    q = cache.queries()
    out = cache.tree_attend(ctx, q)
    assert ctx.sync() == 0
    cache.check(ctx, q, out)
    assert ctx.sync() == 0


@pytest.mark.gpu
def test_rows_strides_and_requests_left_out(pcl, torch, ctx):
    # requests without new tokens or rows, rows in another order, padded strides:
    # what no request owns stays as it was
    heads = (4, 2, 64)
    held, counts = [40, 9, 300, 7, 600, 0], [2, 0, 3, 1, 2, 4]
    first = [9, 0, 4, 0, 0, 12]
    cache = TreeCache(pcl, torch, heads, held, counts, 16, "f32", 5, first=first, rows=17)
    cache.newest[4] = -7
    q = torch.randn((17, 4 * 64 + 12), device="cuda:0")
    used = [0, 4, 5, 6, 9, 10, 12, 13, 14, 15]
    rest = [i for i in range(17) if i not in used]
    q[rest] = float("nan")  # rows of no active request are not read
    out = torch.full((17, 4 * 64 + 8), 9.5, device="cuda:0")
    cache.tree_attend(ctx, q, out=out)
    assert ctx.sync() == 0
    assert bool((out[:, 256:] == 9.5).all()) and bool((out[rest] == 9.5).all())
    cache.check(ctx, q, out, requests=[0, 2, 3, 5])
    # nobody: nothing happens
    out.fill_(9.5)
    cache.tree_attend(ctx, q, out=out, requests=0)
    cache.newest.fill_(-1)
    cache.tree_attend(ctx, q, out=out)
    assert ctx.sync() == 0
    assert bool((out == 9.5).all())


@pytest.mark.gpu
def test_device_side_errors(pcl, torch, ctx):
    heads = (4, 2, 64)
    held, counts = [40, 300, 700], [3, 5, 70]
    masks, positions = random_trees(np.random.default_rng(5), held, counts)
    cache = TreeCache(pcl, torch, heads, held, counts, 16, "f32", 6, masks, positions)
    q = cache.queries()
    good = cache.tree_attend(ctx, q)
    assert ctx.sync() == 0
    mine = [slice(f, f + n) for f, n in zip(cache.first, counts)]

    def left_out(out, b):
        assert bool((out[mine[b]] == 9.5).all())
        assert all(torch.equal(out[mine[i]], good[mine[i]]) for i in range(3) if i != b)

    # lengths, counts and rows out of range
    for name, bad, b in (("dheld", -1, 1), ("dheld", 306, 1), ("dheld", 200, 1),
                         ("dlengths", 1 << 30, 1), ("dlengths", -5, 1), ("newest", 3, 1),
                         ("newest", cache.rows, 2), ("newest", (1 << 31) - 1, 2)):
        x = getattr(cache, name)
        old = x.clone()
        x[b] = bad
        out = cache.tree_attend(ctx, q)
        assert ctx.sync() == BAD_PAGES, (name, bad)
        left_out(out, b)
        x.copy_(old)
    out = cache.tree_attend(ctx, q, max_new=69)
    assert ctx.sync() == BAD_PAGES
    left_out(out, 2)
    out = cache.tree_attend(ctx, q, max_length=769)
    assert ctx.sync() == BAD_PAGES
    left_out(out, 2)
    # more new tokens than the masks have bits
    keep = cache.dmasks
    cache.dmasks, cache.words = keep[:, :1].contiguous(), 1
    out = cache.tree_attend(ctx, q)
    assert ctx.sync() == BAD_PAGES
    left_out(out, 2)
    cache.dmasks, cache.words = keep, 2
    # every request over the same rows: within bounds, whatever comes of it
    newest = cache.newest.clone()
    cache.newest.fill_(75)
    cache.tree_attend(ctx, q)
    assert ctx.sync() == 0
    cache.newest.copy_(newest)
    # pages outside the pools are reported and read as page 0
    table = cache.table.clone()
    cache.pools.k[0] = 1.0
    cache.pools.v[0] = 1.0
    good = cache.tree_attend(ctx, q)
    assert ctx.sync() == 0
    for bad in (cache.pools.k.shape[0], -1, (1 << 31) - 1, -(1 << 31)):
        cache.table[1, 3] = bad
        out = cache.tree_attend(ctx, q)
        assert ctx.sync() == BAD_PAGES
        assert all(torch.equal(out[mine[i]], good[mine[i]]) for i in (0, 2))
        cache.table.copy_(table)
    # a NaN in an attended key or value is reported
    slot = int(cache.table[2, 0]) * 16 + 3
    for x, bit in ((cache.pools.k, 1), (cache.pools.v, 2)):
        flat = x.view(-1, 2, 64)
        old = flat[slot].clone()
        flat[slot, 1, 5] = float("nan")
        cache.tree_attend(ctx, q)
        assert ctx.sync() & bit
        inside = cache.tree_attend(ctx, q, window=600)
        assert ctx.sync() == 0 and bool(torch.isfinite(inside).all())
        flat[slot] = old


@pytest.mark.gpu
def test_slots_past_32_bit_offsets(pcl, torch, ctx):
    kvheads, dim, page = 8, 256, 64
    pages = (1 << 31) // (page * kvheads * dim) + 40
    k = torch.empty((pages, page, kvheads, dim), device="cuda:0", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    pools = pcl.page_pools(k=k.data_ptr(), v=v.data_ptr(), type=pcl.CACHE_BF16, pages=pages,
                           page_tokens=page, kvheads=kvheads, dim=dim)
    for new in (5, 40):  # a few rows, many rows
        held = 300 - new
        cache = TreeCache(pcl, torch, (16, 8, 256), [held], [new], page, "bf16", 3)
        table = torch.tensor([[pages - 1, 2, pages - 3, pages - 2, pages - 7]],
                             dtype=torch.int32, device="cuda:0")
        position = torch.arange(300, device="cuda:0")
        slots = (table[0, position // page] * page + position % page).int()
        ctx.paged_append(pools, slots.data_ptr(), cache.k[0].data_ptr(), cache.v[0].data_ptr(),
                         300)
        q = cache.queries()
        out = cache.tree_attend(ctx, q, pools=pools, table=table.data_ptr(), table_stride=5,
                                max_length=320)
        assert ctx.sync() == 0
        cache.check(ctx, q, out)


@pytest.mark.gpu
def test_many_requests(pcl, torch, ctx):
    rng = np.random.default_rng(4)
    held = [int(n) for n in rng.integers(0, 40, 2048)]
    counts = [int(n) for n in rng.integers(0, 4, 2048)]
    held[7], held[2047], held[1000] = 600, 258, 1025
    counts[7], counts[2047], counts[1000] = 9, 1, 20
    cache = TreeCache(pcl, torch, (2, 1, 64), held, counts, 16, "f32", 12)
    q = cache.queries()
    out = cache.tree_attend(ctx, q)
    assert ctx.sync() == 0
    cache.check(ctx, q, out, exact=False,
                requests=[0, 1, 7, 500, 999, 1000, 1001, 2046, 2047] + list(range(40, 80)))


# Launches whose first spans of 16 chunks are items: those have at least as many chunks
# (over units of 16, 32, 48 or 64 rows and KV heads) as one span for each of 256 CUs'
# workgroups. Requests of one span, of a whole and a part, and of several with single
# chunks behind; a request without new tokens among them.
@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype,held,counts,window", [
    ((16, 8, 256), "bf16", [1900, 200, 0, 5000], [700, 500, 0, 129], 0),
    ((16, 8, 256), "f32", [30, 9000], [3, 400], 0),
    ((16, 8, 256), "bf16", [15000, 4090], [700, 16], 0),
    ((16, 8, 256), "f32", [20000, 600], [700, 500], 4200),
    ((16, 2, 512), "f32", [9000, 8190, 8000, 100, 10000, 7000], [64, 80, 64, 3, 64, 70], 0),
    ((10, 2, 208), "bf16", [9000, 16000, 4000], [300, 400, 100], 0),
    ((16, 4, 64), "f32", [100 + i for i in range(12)], [600] * 12, 0),
], ids=str)
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_spans_as_items(pcl, torch, ctx, heads, dtype, held, counts, window, tree):
    counts = [min(n, 500) for n in counts] if tree else counts
    masks = positions = None
    if tree:
        masks, positions = random_trees(np.random.default_rng(19), held, counts)
    cache = TreeCache(pcl, torch, heads, held, counts, 64, dtype, 23, masks, positions)
    q = cache.queries()
    out = cache.tree_attend(ctx, q, window=window)
    assert ctx.sync() == 0
    again = cache.tree_attend(ctx, q, window=window)
    assert np.array_equal(bits(out), bits(again))
    cache.check(ctx, q, out, window=window, exact=False)
    assert ctx.sync() == 0


@pytest.mark.gpu
def test_replays_over_other_requests(pcl, torch):
    # one capture, each replay with other requests taking part: launches whose spans are
    # items and launches of single chunks, in turn, on a stream of their own
    heads, held, counts = (16, 8, 256), [9000, 500, 15000, 40], [400, 70, 300, 9]
    stream = torch.cuda.Stream()
    cache = TreeCache(pcl, torch, heads, held, counts, 16, "bf16", 31)
    q = cache.queries()
    out = torch.full_like(q, 9.5)
    newest = cache.newest.clone()
    torch.cuda.synchronize()
    own = pcl.Context(0, stream.cuda_stream)
    d = cache.tree_desc(own, q, out)
    own.reserve(own.paged_tree_workspace_bytes(d))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.paged_tree_attention(d)
    eager = pcl.Context(0)
    whole = cache.tree_attend(eager, q)
    cache.check(eager, q, whole, exact=False)
    for taking in ([0, 1, 2, 3], [1, 3], [2], [], [0, 2], [3]):
        cache.newest.fill_(-1)
        cache.newest[taking] = newest[taking]
        out.fill_(9.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.full_like(q, 9.5)
        for b in taking:
            mine = slice(cache.first[b], cache.first[b] + counts[b])
            want[mine] = whole[mine]
        assert np.array_equal(bits(out), bits(want)), taking
        assert np.array_equal(bits(cache.tree_attend(eager, q)), bits(want)), taking
    assert [c.sync() for c in (own, eager)] == [0, 0]
    graph.reset()
    own.close()
    eager.close()


@pytest.mark.gpu
def test_prompts_beside_single_tokens(pcl, torch, ctx):
    # one launch with requests of one new token and of many
    held, counts = [700, 0, 33, 1500, 260, 90], [1, 400, 2, 1, 150, 17]
    for heads, dtype in (((16, 8, 256), "bf16"), ((16, 2, 512), "f32"), ((6, 2, 112), "f32")):
        cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, 9)
        q = cache.queries()
        out = cache.tree_attend(ctx, q)
        assert ctx.sync() == 0
        cache.check(ctx, q, out)


@pytest.mark.gpu
def test_one_token_equals_the_newest_tokens_attention(pcl, torch, ctx):
    # with one new token each, the bits of pcl_paged_attention
    held = [0, 5, 300, 2000]
    for heads, dtype in (((16, 8, 256), "bf16"), ((4, 2, 64), "f32")):
        cache = TreeCache(pcl, torch, heads, held, [1] * 4, 16, dtype, 9)
        q = cache.queries()
        for window in (0, 200):
            out = cache.tree_attend(ctx, q, window=window)
            other = cache.attend(ctx, q, rows=[0, 1, 2, 3], window=window)
            assert np.array_equal(bits(out + 0.0), bits(other + 0.0))
    assert ctx.sync() == 0


@pytest.mark.gpu
def test_timing_counts_the_launches(pcl, torch):
    own = pcl.Context(0)
    cache = TreeCache(pcl, torch, (4, 2, 64), [700, 40], [3, 3], 16, "f32", 22)
    q = cache.queries()
    cache.tree_attend(own, q)
    own.set_timing(True)
    cache.tree_attend(own, q)
    assert own.sync() == 0
    ms, launches = own.timing()
    assert launches == (1, 1) and ms[0] > 0 and ms[1] > 0
    own.close()


@pytest.mark.gpu
def test_two_contexts_at_once(pcl, torch):
    # each has its stream, workspace and error flag; the pages are shared
    heads = (16, 8, 256)
    caches = [TreeCache(pcl, torch, heads, [3000] * 6, [n] * 6, 16, "bf16", 23) for n in (4, 30)]
    qs = [c.queries(seed=i) for i, c in enumerate(caches)]
    outs = [torch.zeros_like(q) for q in qs]
    own = [pcl.Context(0) for _ in qs]
    descs = [c.tree_desc(x, q, o) for c, x, q, o in zip(caches, own, qs, outs)]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, d in zip(own, descs):
            c.paged_tree_attention(d)
    assert [c.sync() for c in own] == [0, 0]
    for cache, c, q, o in zip(caches, own, qs, outs):
        cache.check(c, q, o, requests=(0, 5), exact=False)
        assert c.sync() == 0
        c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype,counts", [((12, 1, 128), "bf16", [2, 1, 0]),
                                                ((8, 1, 256), "f32", [4, 30, 9]),
                                                ((9, 3, 112), "bf16", [3, 1, 40])], ids=str)
def test_a_first_call_inside_a_capture(pcl, torch, heads, dtype, counts):
    stream = torch.cuda.Stream()
    held = [300, 5, 900]
    masks, positions = random_trees(np.random.default_rng(5), held, counts)
    cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, 9, masks, positions)
    q = cache.queries()
    out = torch.full_like(q, 9.5)
    torch.cuda.synchronize()
    ctx = pcl.Context(0, stream.cuda_stream)
    d = cache.tree_desc(ctx, q, out, max_new=64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        q.mul_(1.0)  # the capture holds a node either way
        with pytest.raises(pcl.AttentionError) as e:
            ctx.paged_tree_attention(d)
        assert e.value.kind == "ResourceLimit"
    torch.cuda.synchronize()
    graph.reset()
    ctx.reserve(ctx.paged_tree_workspace_bytes(d))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.paged_tree_attention(d)
    for i in range(4):
        q.normal_()
        out.fill_(9.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        cache.check(ctx, q, out, exact=False)
        assert ctx.sync() == 0
    graph.reset()
    ctx.close()


# ---- runs of them together ---------------------------------------------------------------

class Drafts:
    """One layer of a batched decoder that verifies drafted trees: the step's raw
    projections through the head transform into the pages at the trees' positions,
    and every new token's attention."""

    def __init__(self, pcl, torch, ctx, heads, shape, window, dtype, words=1):
        requests, stride, page, pages, rows = shape
        qheads, kvheads, dim = heads
        self.torch, self.ctx, self.heads, self.rows = torch, ctx, heads, rows
        self.trees = Trees(pcl, torch, ctx, shape, words)
        self.batch = self.trees.batch
        self.pools = Pools(pcl, torch, pages, page, kvheads, dim, dtype)
        self.limit = stride * page
        scale = 1.0 + 0.1 * np.random.default_rng(0).standard_normal(dim)
        self.transform = pcl.HeadTransform(ctx, qheads, kvheads, dim, scale, scale[::-1], 1e-6,
                                           10000.0)
        dev = {"device": "cuda:0"}
        self.raw = [torch.zeros((rows, h, dim), **dev) for h in (qheads, kvheads, kvheads)]
        self.q = torch.zeros((rows, qheads * dim), **dev)
        self.out = torch.zeros((rows, qheads * dim), **dev)
        a = self.batch.a
        self.desc = ctx.paged_tree_desc(
            pools=self.pools.desc, q=self.q.data_ptr(), q_stride=qheads * dim, q_rows=rows,
            qheads=qheads, table=a["table"].data_ptr(), table_stride=stride,
            lengths=a["lengths"].data_ptr(), step_lengths=a["step_lengths"].data_ptr(),
            newest=a["newest"].data_ptr(), masks=self.trees.masks.data_ptr(), mask_words=words,
            positions=self.trees.positions.data_ptr(), requests=requests, max_length=self.limit,
            max_new=64 * words, window=window, q_scale=scale_of(dim), out=self.out.data_ptr(),
            o_stride=qheads * dim)
        ctx.reserve(ctx.paged_tree_workspace_bytes(self.desc))
        self.depth = 12
        self.paths = torch.zeros((requests, self.depth), dtype=torch.int32, **dev)
        self.kept = torch.zeros(requests, dtype=torch.int32, **dev)
        self.moves = [torch.zeros_like(self.paths) for _ in range(2)]
        ctx.page_reset(self.batch.desc)

    def verify(self):
        """A step's rows, trees and attention."""
        a, ctx = self.batch.a, self.ctx
        ctx.page_step(self.batch.desc, self.batch.words.data_ptr())
        ctx.page_tree(self.batch.desc, self.trees.tree)
        self.transform.append_paged(self.pools.desc, a["slots"].data_ptr(),
                                    self.trees.positions.data_ptr(), self.limit,
                                    *[x.data_ptr() for x in self.raw], self.rows,
                                    self.q.data_ptr())
        ctx.paged_tree_attention(self.desc)

    def keep(self):
        """The verified branches' rows to their places."""
        ctx = self.ctx
        ctx.page_accept(self.batch.desc, self.paths.data_ptr(), self.kept.data_ptr(), self.depth,
                        *[x.data_ptr() for x in self.moves])
        ctx.page_commit(self.batch.desc, self.kept.data_ptr())
        ctx.paged_copy([self.pools.desc], *[x.data_ptr() for x in self.moves],
                       self.kept.shape[0], self.depth)

    def close(self):
        self.transform.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,window,dtype", [((4, 2, 64), 0, "f32"), ((4, 2, 64), 40, "bf16"),
                                                ((2, 1, 256), 40, "f32")],
                         ids=["f32", "window-bf16", "window-d256"])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_rounds_of_drafted_trees(pcl, torch, heads, window, dtype, captured):
    # what a round leaves in the pages, and what the next tokens see, is what the
    # kept tokens decoded one at a time leave; with a graph every round is a replay
    # of two captures
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx = pcl.Context(0, stream.cuda_stream)
    shape = (5, 40, 8, 150, 300)
    run = Drafts(pcl, torch, ctx, heads, shape, window, dtype)
    single = tp.Server(pcl, torch, ctx, heads, shape[0], shape[2], shape[3], shape[1], shape[4],
                       window, dtype)
    model = ShareModel(*shape)
    torch.cuda.synchronize()
    graphs = []
    if captured:
        run.verify()  # no tokens: builds the rotation table
        run.keep()
        torch.cuda.synchronize()
        for part in (run.verify, run.keep):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                part()
            graphs.append(graph)
    parts = [g.replay for g in graphs] or [run.verify, run.keep]
    rng = np.random.default_rng(8)
    g = torch.Generator(device="cuda:0")
    g.manual_seed(3)
    qheads, kvheads, dim = heads
    for counts in ([60, 0, 7, 1, 0], [9, 0, 12, 30, 1], [1, 64, 0, 5, 20], [16, 16, 16, 16, 16]):
        for x in run.raw:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda:0"))
        parents = [random_parents(rng, n) for n in counts]
        branches = [tree_of(p)[1] for p in parents]
        paths = [sorted(b[int(rng.integers(len(b)))])[:run.depth] if b else [] for b in branches]
        run.trees.put(parents)
        run.batch.put(counts)
        run.kept.copy_(torch.tensor([len(p) for p in paths], dtype=torch.int32))
        for b, p in enumerate(paths):
            run.paths[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        run.out.fill_(9.5)
        torch.cuda.synchronize()
        parts[0]()
        torch.cuda.synchronize()
        assert ctx.sync() == 0
        assert model.step(counts)
        out = run.out.clone()
        assert bool((out[sum(counts):] == 9.5).all())
        first = np.concatenate(([0], np.cumsum(counts)))
        # the same tokens through the single-token path, along each branch
        lens = [len(p) for p in paths]
        for k in range(max(lens)):
            now = [int(k < n) for n in lens]
            row = 0
            for b, p in enumerate(paths):
                if now[b]:
                    for x, y in zip(single.raw, run.raw):
                        x[row].copy_(y[int(first[b]) + p[k]])
                    row += 1
            single.batch.put(now)
            torch.cuda.synchronize()
            single.step()
            torch.cuda.synchronize()
            assert ctx.sync() == 0
            row = 0
            for b, p in enumerate(paths):
                if now[b]:
                    # a branch that is the first tokens of its request: the same keys
                    # at the same places, the same bits. Others in other sums.
                    got, want = out[int(first[b]) + p[k]], single.attended[row]
                    if p[:k + 1] == list(range(k + 1)):
                        assert np.array_equal(bits(got + 0.0), bits(want + 0.0))
                    size = float(run.pools.v[run.pools.v == run.pools.v].abs().max())
                    close = 4 * size * (2 * dim * 25 + 2 * 400 + 64) * 2.0 ** -24
                    assert float((got - want).abs().max()) <= close
                    row += 1
        parts[1]()
        torch.cuda.synchronize()
        assert ctx.sync() == 0
        assert model.commit(lens)
        model.check(run.batch.state())
        # the pages hold the kept tokens' rows, as the single tokens' do
        state, other = run.batch.state(), single.batch.state()
        assert state["lengths"].tolist() == other["lengths"].tolist()
        for b, n in enumerate(model.lengths):
            at = np.arange(n)
            slots = [x["table"].reshape(shape[0], -1)[b, at // 8] * 8 + at % 8
                     for x in (state, other)]
            rows = [p.rows(torch.from_numpy(s.astype(np.int64)).to("cuda:0"))
                    for p, s in zip((run.pools, single.pools), slots)]
            for x, y in zip(*rows):
                assert np.array_equal(bits(x), bits(y))
    for graph in graphs:
        graph.reset()
    run.close()
    single.transform.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_answers_that_share_a_prompt(pcl, torch, captured):
    # a prompt, copies of it that go on differently, and their pages given back:
    # every answer attends as one that was prompted by itself
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx = pcl.Context(0, stream.cuda_stream)
    heads, shape, dtype = (4, 2, 64), (6, 12, 8, 40, 200), "f32"
    run = Drafts(pcl, torch, ctx, heads, shape, 0, dtype, words=2)
    layers = [run.pools] + layers_of(pcl, torch, shape[3], shape[2],
                                     [(1, 32, "bf16"), (2, 64, "f32")], 4)
    model = ShareModel(*shape)
    dev = {"dtype": torch.int32, "device": "cuda:0"}
    sources = torch.full((6,), -1, **dev)
    moves = [torch.zeros(6, **dev) for _ in range(3)]
    finished = torch.zeros(6, **dev)
    chain = torch.arange(-1, shape[4] - 1, **dev)

    def step():
        ctx.page_step(run.batch.desc, run.batch.words.data_ptr())
        run.transform.append_paged(run.pools.desc, run.batch.a["slots"].data_ptr(),
                                   run.batch.a["positions"].data_ptr(), run.limit,
                                   *[x.data_ptr() for x in run.raw], run.rows, run.q.data_ptr())
        ctx.paged_tree_attention(run.desc)
        ctx.page_commit(run.batch.desc)

    def fork():
        ctx.page_fork(run.batch.desc, sources.data_ptr(), *[x.data_ptr() for x in moves])
        ctx.page_commit(run.batch.desc)
        ctx.paged_copy([p.desc for p in layers], moves[0].data_ptr(), moves[1].data_ptr(), 6, 1,
                       moves[2].data_ptr())

    def release():
        ctx.page_release_shared(run.batch.desc, finished.data_ptr())

    run.desc.masks, run.desc.mask_words, run.desc.positions = None, 0, None
    parts = [step, fork, release]
    ctx.reserve(max(ctx.paged_tree_workspace_bytes(run.desc),
                    ctx.page_release_workspace_bytes(run.batch.desc)))
    graphs = []
    if captured:
        step()
        torch.cuda.synchronize()
        for i, part in enumerate(parts):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                part()
            graphs.append(graph)
            parts[i] = graph.replay
    history = [[] for _ in range(6)]
    g = torch.Generator(device="cuda:0")
    g.manual_seed(3)
    qheads, kvheads, dim = heads
    plan = [("step", [21, 0, 0, 0, 11, 0]), ("fork", [-1, 0, 0, 4, -1, -1]),
            ("step", [1, 1, 1, 1, 1, 0]), ("step", [3, 9, 1, 30, 1, 2]),
            ("release", [1, 0, 0, 0, 1, 0]), ("fork", [1, -1, -1, -1, 3, -1]),
            ("step", [5, 1, 1, 1, 4, 1]), ("release", [0, 1, 1, 1, 0, 0]),
            ("step", [1, 20, 0, 0, 1, 1])]
    for name, words in plan:
        if name == "step":
            for x in run.raw:
                x.copy_(torch.randn(x.shape, generator=g, device="cuda:0"))
            run.batch.put(words)
            torch.cuda.synchronize()
            parts[0]()
            torch.cuda.synchronize()
            assert model.step(words) and model.commit()
            row = 0
            for b, n in enumerate(words):
                for i in range(n):
                    history[b].append([x[row + i].clone() for x in run.raw])
                if n:
                    raw = [torch.stack([r[i] for r in history[b]]) for i in range(3)]
                    q, k, v = (torch.empty_like(x) for x in raw)
                    total = len(history[b])
                    out = torch.empty((n, qheads * dim), device="cuda:0")
                    torch.cuda.synchronize()
                    run.transform.prepare(*[x.data_ptr() for x in raw], total, 0,
                                          *[x.data_ptr() for x in (q, k, v)])
                    ctx.launch(ctx.desc(
                        q=q[total - n].data_ptr(), q_stride=qheads * dim, nq=n, k0=k.data_ptr(),
                        v0=v.data_ptr(), n0=total, qheads=qheads, kvheads=kvheads, dim=dim,
                        kh_first=0, kh_end=kvheads, causal=1, first_query=total - n,
                        q_scale=scale_of(dim), out=out.data_ptr(), o_stride=qheads * dim))
                    torch.cuda.synchronize()
                    assert np.array_equal(bits(run.out[row:row + n] + 0.0), bits(out + 0.0)), b
                row += n
        elif name == "fork":
            sources.copy_(torch.tensor(words, **dev))
            before = [[x.view(-1, *x.shape[2:]).clone() for x in (p.k, p.v)] for p in layers]
            torch.cuda.synchronize()
            parts[1]()
            torch.cuda.synchronize()
            want = model.fork(words)
            assert want and model.commit()
            assert [x.tolist() for x in moves] == want
            runs = [[(a, b, n)] for a, b, n in zip(*want)]
            for p, old in zip(layers, before):
                for x, y in zip((p.k, p.v), old):
                    now = copy_model(y, runs)
                    same = (x.view(now.shape) == now) | (now != now)
                    assert bool(same.all())
            for b, s in enumerate(words):
                if s >= 0:
                    history[b] = list(history[s])
        else:
            finished.copy_(torch.tensor(words, **dev))
            torch.cuda.synchronize()
            parts[2]()
            torch.cuda.synchronize()
            model.release_shared(words)
            for b, f in enumerate(words):
                if f:
                    history[b] = []
        assert ctx.sync() == 0, (name, words)
        state = run.batch.state()
        assert state["lengths"].tolist() == model.lengths
        assert state["free_pages"][:len(model.free)].tolist() == model.free
        assert state["counters"][0] == len(model.free)
    del chain
    for graph in graphs:
        graph.reset()
    run.close()
    ctx.close()
