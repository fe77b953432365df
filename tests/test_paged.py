"""Batches of requests over a paged cache (pcl_page_*, pcl_paged_*).

Page bookkeeping is checked word for word against a model that handles one
request after another; appended rows bit for bit against their sources
(rounded to bf16 where the pages hold it); transformed rows bit for bit against
the head transform of one token at a time; attention bit for bit against
pcl_attention_launch over each request's rows laid out in one segment, and
against a plain softmax in 64 bits. The run at the end takes a batch through
prompts, decode steps, refused speculative tokens, a release and its reuse.
"""
import ctypes

import numpy as np
import pytest

BAD_PAGES = 32
STATE = ("lengths", "table", "free_pages", "counters", "step_lengths", "newest", "slots",
         "positions", "row_request")


class PageModel:
    """The bookkeeping of a batch, one request after another."""

    def __init__(self, requests, stride, page, pages, rows):
        self.requests, self.stride, self.page = requests, stride, page
        self.pages, self.rows = pages, rows
        self.lengths = [0] * requests
        self.table = [[-1] * stride for _ in range(requests)]
        self.free = [pages - 1 - i for i in range(pages)]
        self.standing = None
        self.void()

    def void(self):
        self.step_lengths = list(self.lengths)
        self.newest = [-1] * self.requests
        self.slots, self.positions, self.row_request = [], [], []
        self.taken = 0

    def held(self, tokens):
        return -(-tokens // self.page)

    def step(self, counts):
        """False when the step is refused."""
        self.void()
        self.standing = None
        cap = self.stride * self.page
        need = 0
        for n, c in zip(self.lengths, counts):
            if n < 0 or n > cap or c < 0 or n + c > cap:
                return False
            need += self.held(n + c) - self.held(n)
        if need > len(self.free) or sum(counts) > self.rows:
            return False
        for b, c in enumerate(counts):
            n = self.lengths[b]
            for p in range(n, n + c):
                column = p // self.page
                if column >= self.held(n) and p % self.page == 0:
                    self.table[b][column] = self.free[len(self.free) - 1 - self.taken]
                    self.taken += 1
                self.slots.append(self.table[b][column] * self.page + p % self.page)
                self.positions.append(p)
                self.row_request.append(b)
            if c:
                self.newest[b] = len(self.slots) - 1
            self.step_lengths[b] = n + c
        self.standing = list(counts)
        return True

    def give_back(self, before, after):
        for b in range(self.requests):
            for column in range(self.held(after[b]), self.held(before[b])):
                self.free.append(self.table[b][column])
        self.lengths = list(after)

    def commit(self, kept=None):
        """False when the call is refused."""
        if self.standing is None:
            return True
        kept = self.standing if kept is None else kept
        if any(k < 0 or k > c for k, c in zip(kept, self.standing)):
            return False
        if self.taken:
            del self.free[-self.taken:]
        self.give_back(self.step_lengths, [n + k for n, k in zip(self.lengths, kept)])
        self.standing = None
        return True

    def release(self, finished):
        self.give_back(self.lengths, [0 if f else n for n, f in zip(self.lengths, finished)])
        self.standing = None

    def check(self, state):
        """`state`: the arrays by name, as numpy arrays."""
        n = len(self.slots)
        assert state["lengths"].tolist() == self.lengths
        assert state["counters"][0] == len(self.free)
        assert state["counters"][3] == (self.standing is not None)
        assert state["free_pages"][:len(self.free)].tolist() == self.free
        assert state["table"].reshape(self.requests, -1).tolist() == self.table
        assert state["step_lengths"].tolist() == self.step_lengths
        assert state["newest"].tolist() == self.newest
        for name in ("slots", "positions", "row_request"):
            assert state[name].tolist() == getattr(self, name) + [-1] * (self.rows - n), name
        assert state["counters"][1] == n


# (requests, table stride, tokens a page, pages, rows): one request, odd page
# sizes, pages of one token, more requests than the workgroup has threads, steps
# of several workgroups
BATCHES = [(1, 4, 16, 6, 70), (3, 9, 7, 20, 130), (5, 40, 1, 90, 64), (37, 6, 16, 120, 700),
           (300, 3, 8, 500, 900), (2048, 2, 4, 2600, 2500)]


def drive(model, call, seed, steps=25):
    """A random run of steps, commits and releases, some of them refused;
    call(name, words) runs one on the other side and returns (error, state)."""
    rng = np.random.default_rng(seed)
    refused = 0
    for _ in range(steps):
        room = [model.stride * model.page - n for n in model.lengths]
        counts = [int(min(r, c)) for r, c in zip(room, rng.choice(
            [0, 1, 1, 1, 2, model.page, 3 * model.page + 1], model.requests))]
        budget = model.rows  # most steps fit: later requests take less
        if rng.random() < 0.8:
            for b in range(model.requests):
                counts[b] = min(counts[b], max(0, budget))
                budget -= counts[b]
        if rng.random() < 0.1:
            counts[int(rng.integers(model.requests))] = int(rng.choice([-1, 1 << 30]))
        ok = model.step(counts)
        refused += not ok
        error, state = call("step", counts)
        assert error == (0 if ok else BAD_PAGES)
        model.check(state)
        kind = rng.random()
        if kind < 0.55:
            error, state = call("commit", None)
            assert model.commit() and error == 0
        elif kind < 0.8:
            kept = [int(rng.integers(0, max(c, 0) + 1)) for c in counts]
            if rng.random() < 0.2:
                kept[-1] = int(rng.choice([-1, 1 << 20]))
            good = model.commit(kept)
            error, state = call("commit", kept)
            assert error == (0 if good else BAD_PAGES)
        if rng.random() < 0.3 or len(model.free) < model.pages // 4:
            finished = [int(f) for f in rng.integers(0, 2, model.requests)]
            model.release(finished)
            error, state = call("release", finished)
            assert error == 0
        # what a step wrote stands until the next step
        state = dict(state)
        n = len(model.slots)
        assert state["slots"][:n].tolist() == model.slots
        model.check(state)
    return refused


def test_the_model_itself():
    m = PageModel(2, 3, 4, 5, 16)
    assert m.step([5, 0]) and m.slots == [0, 1, 2, 3, 4] and m.newest == [4, -1]
    assert m.table[0][:2] == [0, 1] and m.taken == 2
    assert m.commit([4, 0]) and m.free == [4, 3, 2, 1] and m.lengths == [4, 0]
    assert m.step([1, 9]) and m.slots[0] == 1 * 4
    assert m.positions == [4] + list(range(9)) and m.taken == 4
    assert m.commit() and m.free == []
    assert not m.step([4, 0]) and m.slots == []  # no page left
    assert not m.step([0, 4])  # past the table
    m.release([0, 1])
    assert m.free == [2, 3, 4] and m.lengths == [5, 0]


# ---- refusals (no device work) ----------------------------------------------

def batch_of(pcl, **kw):
    fields = dict(requests=2, table_stride=4, page_tokens=16, pages=8, step_rows=32)
    fields.update({n: 64 for n in STATE})
    fields.update(kw)
    return pcl.page_batch(**fields)


def pools_of(pcl, **kw):
    fields = dict(k=64, v=64, type=pcl.CACHE_F32, pages=8, page_tokens=16, kvheads=2, dim=64)
    fields.update(kw)
    return pcl.page_pools(**fields)


def paged_of(pcl, pools=None, **kw):
    fields = dict(q=64, q_stride=256, q_rows=2, qheads=4, table=64, table_stride=4, lengths=64,
                  rows=64, requests=2, max_length=64, out=64, o_stride=256)
    fields.update(kw)
    return pcl.Context.paged_desc(pools=pools or pools_of(pcl), **fields)


@pytest.fixture()
def no_context():
    """Memory that stands in for a context: a refused call reads none of it."""
    return ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)


@pytest.mark.parametrize("kw", [
    dict(requests=0), dict(requests=-1), dict(requests=2049), dict(table_stride=0),
    dict(table_stride=1 << 40), dict(page_tokens=0), dict(page_tokens=4097), dict(pages=0),
    dict(pages=1 << 27), dict(step_rows=0), dict(step_rows=1 << 20)] +
    [{n: None} for n in STATE] + [{n: 66} for n in STATE], ids=str)
def test_page_calls_refuse_bad_batches(pcl, no_context, kw):
    lib = pcl.load()
    b = ctypes.byref(batch_of(pcl, **kw))
    words = ctypes.c_void_p(64)
    assert lib.pcl_page_reset(no_context, b) == pcl.INVALID_SHAPE
    assert lib.pcl_page_step(no_context, b, words) == pcl.INVALID_SHAPE
    assert lib.pcl_page_commit(no_context, b, None) == pcl.INVALID_SHAPE
    assert lib.pcl_page_release(no_context, b, words) == pcl.INVALID_SHAPE


def test_page_calls_refuse_missing_words(pcl, no_context):
    lib = pcl.load()
    b = ctypes.byref(batch_of(pcl))
    for words in (None, ctypes.c_void_p(66)):
        assert lib.pcl_page_step(no_context, b, words) == pcl.INVALID_SHAPE
        assert lib.pcl_page_release(no_context, b, words) == pcl.INVALID_SHAPE
    assert lib.pcl_page_commit(no_context, b, ctypes.c_void_p(66)) == pcl.INVALID_SHAPE
    for fn in (lib.pcl_page_reset, lib.pcl_page_commit):
        args = (b,) if fn is lib.pcl_page_reset else (b, None)
        assert fn(None, *args) == pcl.INVALID_SHAPE
    assert lib.pcl_page_reset(no_context, None) == pcl.INVALID_SHAPE


BAD_POOLS = [dict(k=None), dict(v=None), dict(k=72), dict(v=68), dict(type=2), dict(type=-1),
             dict(pages=0), dict(pages=1 << 28), dict(page_tokens=0), dict(page_tokens=4097),
             dict(kvheads=0), dict(kvheads=4097), dict(dim=0), dict(dim=24), dict(dim=528)]


@pytest.mark.parametrize("kw", BAD_POOLS, ids=str)
def test_appends_and_attention_refuse_bad_pools(pcl, no_context, kw):
    lib = pcl.load()
    pools = pools_of(pcl, **kw)
    p = ctypes.c_void_p(64)
    assert lib.pcl_paged_append(no_context, ctypes.byref(pools), p, p, p, 1) == pcl.INVALID_SHAPE
    d = paged_of(pcl, pools)
    assert lib.pcl_paged_attention(no_context, ctypes.byref(d)) == pcl.INVALID_SHAPE
    assert lib.pcl_paged_workspace_bytes(ctypes.byref(d)) == 0


def test_append_refuses_bad_rows(pcl, no_context):
    lib = pcl.load()
    pools = ctypes.byref(pools_of(pcl))
    p, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)
    good = (p, p, p, 1)
    for args in ((None, p, p, 1), (p, None, p, 1), (p, p, None, 1), (ctypes.c_void_p(66), p, p, 1),
                 (p, odd, p, 1), (p, p, odd, 1), (p, p, p, -1), (p, p, p, 1 << 20)):
        assert lib.pcl_paged_append(no_context, pools, *args) == pcl.INVALID_SHAPE
    assert lib.pcl_paged_append(None, pools, *good) == pcl.INVALID_SHAPE
    assert lib.pcl_paged_append(no_context, None, *good) == pcl.INVALID_SHAPE
    assert lib.pcl_paged_append(no_context, pools, None, None, None, 0) == pcl.OK
    assert lib.pcl_paged_append_transformed(None, pools, p, p, 8, p, p, p, 1, p) == \
        pcl.INVALID_SHAPE


@pytest.mark.parametrize("kw,code", [
    (dict(qheads=0), 1), (dict(qheads=3), 1), (dict(qheads=4098), 1), (dict(requests=-1), 1),
    (dict(requests=2049), 1), (dict(window=-1), 1), (dict(q=None), 1), (dict(out=None), 1),
    (dict(table=None), 1), (dict(lengths=None), 1), (dict(table_stride=0), 1),
    (dict(max_length=0), 1), (dict(max_length=65), 1), (dict(q_rows=0), 1),
    (dict(rows=None, q_rows=1), 1), (dict(q_stride=252), 1), (dict(q_stride=258), 1),
    (dict(o_stride=252), 1), (dict(o_stride=257), 1), (dict(q=72), 1), (dict(out=72), 1),
    (dict(table=66), 1), (dict(lengths=66), 1), (dict(rows=66), 1), (dict(softcap=-1.0), 2),
    (dict(softcap=float("nan")), 2), (dict(softcap=float("inf")), 2), (dict(softcap=1e-40), 2),
    (dict(softcap=2.0 ** 127), 2), (dict(q_scale=float("nan")), 2),
    (dict(q_scale=float("inf")), 2),
    (dict(requests=2048, q_rows=2048, max_length=1 << 30, table_stride=1 << 30), 1)], ids=str)
def test_attention_refuses_bad_descriptors(pcl, no_context, kw, code):
    lib = pcl.load()
    d = paged_of(pcl, **kw)
    assert lib.pcl_paged_attention(no_context, ctypes.byref(d)) == code
    assert lib.pcl_paged_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.pcl_paged_attention(None, ctypes.byref(paged_of(pcl))) == 1
    assert lib.pcl_paged_attention(no_context, None) == 1


def test_workspace_holds_every_chunk_of_every_request(pcl):
    lib = pcl.load()

    def nbytes(**kw):
        return lib.pcl_paged_workspace_bytes(ctypes.byref(paged_of(
            pcl, pools_of(pcl, page_tokens=256, pages=64), table_stride=64, **kw)))

    # no partials while one chunk holds a request
    base = nbytes(max_length=256)
    assert nbytes(max_length=1) == base > 0
    # (dim + 2) floats per query head and chunk
    assert nbytes(max_length=257) - base == 2 * 2 * 4 * 66 * 4
    assert nbytes(max_length=2561) - base == 2 * 11 * 4 * 66 * 4
    # a window's keys lie in at most (window + 254) div 256 + 1 chunks
    assert nbytes(max_length=16384, window=1) == base
    assert nbytes(max_length=16384, window=2) - base == 2 * 2 * 4 * 66 * 4
    assert nbytes(max_length=16384, window=1024) - base == 2 * 5 * 4 * 66 * 4
    assert nbytes(max_length=1000, window=1 << 40) - base == 2 * 4 * 4 * 66 * 4
    assert nbytes(max_length=256, requests=0) == 0


@pytest.mark.parametrize("window", [16384, 1 << 31, (1 << 63) - 255, (1 << 63) - 254,
                                    (1 << 63) - 1])
def test_a_window_past_the_longest_request_is_no_window(pcl, window):
    # the whole range of the argument: the workspace is that of all keys, and so
    # is the bound of the items
    lib = pcl.load()

    def nbytes(window, **kw):
        kw = dict(dict(table_stride=64, max_length=16384), **kw)
        return lib.pcl_paged_workspace_bytes(ctypes.byref(paged_of(
            pcl, pools_of(pcl, page_tokens=256, pages=64), window=window, **kw)))

    for n in (1, 256, 257, 1000, 16384):
        assert nbytes(window, max_length=n) == nbytes(0, max_length=n) > 0
    if window > 1 << 30:
        many = dict(requests=2048, q_rows=2048, max_length=1 << 30, table_stride=1 << 30)
        assert nbytes(window, **many) == nbytes(0, **many) == 0


@pytest.mark.parametrize("source,kernel", [
    # 16/8/256 heads in f32 and bf16 pages: many items, and few
    ("paged_kv_d256.hip", "_ZN3pcl15paged_kv_kernelILi256EfLb1ELi1ELi1EEEvNS_11PagedParamsE"),
    ("paged_kv_d256.hip", "_ZN3pcl15paged_kv_kernelILi256EDF16bLb1ELi1ELi1EEEvNS_11PagedParamsE"),
    ("paged_kv_d256.hip", "_ZN3pcl15paged_kv_kernelILi256EfLb1ELi1ELi2EEEvNS_11PagedParamsE"),
    ("paged_kv_d256.hip", "_ZN3pcl15paged_kv_kernelILi256EfLb1ELi2ELi1EEEvNS_11PagedParamsE"),
    ("paged_attention.hip",
     "_ZN3pcl20paged_combine_kernelILi8EEEvNS_11PagedParamsENS_12CombineShapeE"),
    ("head_transform.hip",
     "_ZN3pcl22paged_transform_kernelILi256ELi16EDF16bEEvNS_15TransformParamsE"),
])
def test_paged_kernels_do_not_spill_registers(source, kernel):
    # the chunk kernel is held to three waves a SIMD: a spill would cost every
    # unit of K and V
    import os
    from test_boundary import _resource_remarks
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc absent")
    spills = _resource_remarks(source)
    assert kernel in spills, sorted(spills)
    assert spills[kernel] == 0


# ---- on the device ----------------------------------------------------------

@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


@pytest.fixture(scope="module")
def ctx(pcl, torch):
    c = pcl.Context(0, torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


class DeviceBatch:
    """Device arrays of a batch and its descriptor."""

    def __init__(self, pcl, torch, requests, stride, page, pages, rows):
        self.torch = torch
        size = {"lengths": requests, "table": requests * stride, "free_pages": pages,
                "counters": 4, "step_lengths": requests, "newest": requests, "slots": rows,
                "positions": rows, "row_request": rows}
        self.a = {n: torch.full((size[n],), 7, dtype=torch.int32, device="cuda:0") for n in STATE}
        self.desc = pcl.page_batch(requests=requests, table_stride=stride, page_tokens=page,
                                   pages=pages, step_rows=rows,
                                   **{n: self.a[n].data_ptr() for n in STATE})
        self.words = torch.zeros(requests, dtype=torch.int32, device="cuda:0")

    def put(self, values):
        self.words.copy_(self.torch.tensor(values, dtype=self.torch.int32))
        return self.words.data_ptr()

    def state(self):
        return {n: x.cpu().numpy() for n, x in self.a.items()}


def device_call(ctx, batch):
    def call(name, values):
        if name == "step":
            ctx.page_step(batch.desc, batch.put(values))
        elif name == "release":
            ctx.page_release(batch.desc, batch.put(values))
        else:
            ctx.page_commit(batch.desc, None if values is None else batch.put(values))
        return ctx.sync(), batch.state()
    return call


@pytest.mark.gpu
@pytest.mark.parametrize("shape", BATCHES, ids=lambda s: "x".join(map(str, s)))
def test_bookkeeping_follows_the_model(pcl, torch, ctx, shape):
    batch = DeviceBatch(pcl, torch, *shape)
    ctx.page_reset(batch.desc)
    model = PageModel(*shape)
    assert ctx.sync() == 0
    model.check(batch.state())
    drive(model, device_call(ctx, batch), sum(shape))


@pytest.mark.gpu
def test_damaged_tables_are_reported(pcl, torch, ctx):
    batch = DeviceBatch(pcl, torch, 2, 4, 8, 6, 40)
    ctx.page_reset(batch.desc)
    ctx.page_step(batch.desc, batch.put([5, 9]))
    ctx.page_commit(batch.desc)
    assert ctx.sync() == 0
    good = batch.state()
    # a page past the pools in a held entry: that row alone has no slot
    for bad in (6, -1, 1 << 30, -(1 << 31)):
        batch.a["table"][0] = bad
        ctx.page_step(batch.desc, batch.put([1, 1]))
        assert ctx.sync() == BAD_PAGES
        assert batch.state()["slots"][:3].tolist() == [-1, good["table"][5] * 8 + 1, -1]
    batch.a["table"].copy_(torch.from_numpy(good["table"]))
    # a page past the pools on the free list; its entry is not written
    top = int(good["counters"][0]) - 1
    batch.a["free_pages"][top] = 99
    ctx.page_step(batch.desc, batch.put([4, 0]))
    assert ctx.sync() == BAD_PAGES
    state = batch.state()
    assert state["slots"][:5].tolist() == [good["table"][0] * 8 + i for i in (5, 6, 7)] + [-1, -1]
    assert np.array_equal(state["table"], good["table"])
    batch.a["free_pages"].copy_(torch.from_numpy(good["free_pages"]))
    # lengths and free counts out of range refuse the whole step
    for name, bad in (("lengths", -1), ("lengths", 33), ("counters", 7), ("counters", -1)):
        batch.a[name][0] = bad
        ctx.page_step(batch.desc, batch.put([0, 1]))
        assert ctx.sync() == BAD_PAGES
        assert batch.state()["counters"][1:].tolist() == [0, 0, 0]
        assert (batch.state()["slots"] == -1).all()
        batch.a[name].copy_(torch.from_numpy(good[name]))
    ctx.page_step(batch.desc, batch.put([1, 1]))
    assert ctx.sync() == 0
    # step lengths that fell below the held ones: the commit changes nothing
    batch.a["step_lengths"][1] = 3
    ctx.page_commit(batch.desc)
    assert ctx.sync() == BAD_PAGES
    assert np.array_equal(batch.state()["lengths"], good["lengths"])


@pytest.mark.gpu
def test_a_step_over_damaged_pages_is_not_committed(pcl, torch, ctx):
    # request 0 held pages 0 and 1, gave them back, and request 1 owns them now:
    # request 0's table still names them
    batch = DeviceBatch(pcl, torch, 2, 4, 8, 6, 20)
    model = PageModel(2, 4, 8, 6, 20)
    call = device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    for name, words in (("step", [9, 0]), ("commit", None), ("release", [1, 0]), ("step", [0, 9]),
                        ("commit", None)):
        getattr(model, name)(*([] if words is None else [words]))
        error, state = call(name, words)
        assert error == 0
        model.check(state)
    assert model.table == [[0, 1, -1, -1], [1, 0, -1, -1]] and model.lengths == [0, 9]
    good = {n: x.clone() for n, x in batch.a.items()}
    top = len(model.free) - 1

    def held():
        return [batch.a[n].cpu().numpy().copy() for n in ("lengths", "counters", "free_pages")]

    # a number outside the pools on the free list: no page of another request
    # stands in its place, the step does not stand, so that nothing of it is
    # committed, and the next step does not find the pages held
    for bad in (6, -1, 99, 1 << 30, -(1 << 31)):
        batch.a["free_pages"][top] = bad
        error, state = call("step", [5, 0])
        assert error == BAD_PAGES and (state["slots"] == -1).all()
        assert state["counters"][3] == 0
        assert state["table"].tolist() == [-1, 1, -1, -1, 1, 0, -1, -1]
        before = held()
        for kept in (None, [5, 0], [2, 0], [0, 0]):
            error, _ = call("commit", kept)
            assert error == 0
            assert all(np.array_equal(x, y) for x, y in zip(before, held()))
        batch.a["free_pages"][top] = good["free_pages"][top]
        error, state = call("step", [5, 1])
        assert error == 0 and state["slots"][:6].tolist() == [8 * 2 + i for i in range(5)] + [1]
        for n, x in good.items():
            batch.a[n].copy_(x)
    # one in a held entry: the partly filled page that the step goes on in, a page
    # that a release gives back
    batch.a["table"][4 + 1] = 6
    error, _ = call("step", [1, 1])
    assert error == BAD_PAGES
    before = held()
    assert before[1][3] == 0 and call("commit", None)[0] == 0
    assert all(np.array_equal(x, y) for x, y in zip(before, held()))
    # (a step that does not touch the page is committed)
    assert call("step", [1, 0])[0] == 0 and call("commit", None)[0] == 0
    before = held()
    assert call("release", [1, 1])[0] == BAD_PAGES
    assert all(np.array_equal(x, y) for x, y in zip(before, held()))
    assert call("release", [1, 0])[0] == 0
    assert batch.a["lengths"].tolist() == [0, 9]
    # or one behind the step among the pages that a commit gives back
    for n, x in good.items():
        batch.a[n].copy_(x)
    assert call("step", [17, 3])[0] == 0
    batch.a["table"][2] = 6
    before = held()
    assert call("commit", [1, 3])[0] == BAD_PAGES
    assert all(np.array_equal(x, y) for x, y in zip(before, held()))


@pytest.mark.gpu
def test_shared_pages_are_not_released(pcl, torch, ctx):
    # block tables may share pages; one that another request holds, or that two
    # requests give back at once, must not come to be free: the release is refused
    shape = (4, 6, 8, 24, 100)
    batch = DeviceBatch(pcl, torch, *shape)
    model = PageModel(*shape)
    call = device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    model.step([20, 30, 9, 5])
    assert call("step", [20, 30, 9, 5])[0] == 0
    model.commit()
    assert call("commit", None)[0] == 0
    model.step([1, 1, 1, 1])
    assert call("step", [1, 1, 1, 1])[0] == 0  # it stands
    good = {n: x.clone() for n, x in batch.a.items()}

    def back():
        for n, x in good.items():
            batch.a[n].copy_(x)

    def refused(finished):
        before = batch.state()
        error, after = call("release", finished)
        assert error == BAD_PAGES
        for n in STATE:
            assert np.array_equal(before[n], after[n]), n

    # request 1 begins with the pages of request 0
    batch.a["table"][6:8] = batch.a["table"][:2]
    for finished in ([1, 0, 0, 0], [0, 1, 0, 0], [1, 1, 0, 0], [1, 1, 1, 1], [0, 1, 0, 7]):
        refused(finished)
    # the others are released as ever, and nobody at all
    assert call("release", [0, 0, 0, 0])[0] == 0
    error, state = call("release", [0, 0, 1, 1])
    assert error == 0 and state["lengths"].tolist() == [20, 30, 0, 0]
    assert state["free_pages"][:int(state["counters"][0])].tolist() == model.free + [7, 8, 9]
    refused([1, 0, 0, 0])
    # each with its own pages again
    batch.a["table"].copy_(good["table"])
    error, state = call("release", [1, 0, 0, 0])
    assert error == 0
    assert state["free_pages"][:int(state["counters"][0])].tolist() == \
        model.free + [7, 8, 9, 0, 1, 2]
    # a page twice in one table
    back()
    batch.a["table"][1] = batch.a["table"][0]
    refused([1, 0, 0, 0])
    # the only page that is shared is the last one of either
    back()
    batch.a["table"][6 + 3] = batch.a["table"][2]
    refused([0, 1, 0, 0])
    # words behind the list may hold anything, words of it may not
    for word in (-1, -(1 << 31), (1 << 31) - 1, 5):
        back()
        batch.a["free_pages"][len(model.free):] = word
        error, state = call("release", [0, 0, 1, 0])
        assert error == 0
        assert state["free_pages"][:int(state["counters"][0])].tolist() == model.free + [7, 8]
        if word < 0:
            back()
            batch.a["free_pages"][3] = word
            refused([0, 0, 1, 0])


@pytest.mark.gpu
def test_one_shared_page_among_many_is_found(pcl, torch, ctx):
    # more words, returned and kept pages than the workgroup's threads take at once
    shape = (40, 700, 1, 20000, 16000)
    batch = DeviceBatch(pcl, torch, *shape)
    model = PageModel(*shape)
    call = device_call(ctx, batch)
    ctx.page_reset(batch.desc)
    counts = [100 + 15 * (b % 41) for b in range(40)]
    assert model.step(counts) and call("step", counts)[0] == 0
    assert model.commit() and call("commit", None)[0] == 0
    finished = [b % 2 for b in range(40)]
    good = batch.a["table"].clone()
    for b, column in ((0, 0), (38, counts[38] - 1), (20, 133)):
        for c, other in ((1, 0), (39, counts[39] - 1), (21, 250)):
            batch.a["table"][700 * b + column] = batch.a["table"][700 * c + other]
            error, state = call("release", finished)
            assert error == BAD_PAGES
            assert state["lengths"].tolist() == counts
            assert state["free_pages"][:len(model.free)].tolist() == model.free
            batch.a["table"].copy_(good)
    model.release(finished)
    error, state = call("release", finished)
    assert error == 0
    model.void()  # (what the step wrote stands)
    for name in ("lengths", "free_pages", "counters"):
        want = {"lengths": model.lengths, "free_pages": model.free,
                "counters": [len(model.free)]}[name]
        assert state[name][:len(want)].tolist() == want
    rest = [1 - f for f in finished]
    model.release(rest)
    error, state = call("release", rest)
    assert error == 0 and len(model.free) == 20000
    assert state["free_pages"].tolist() == model.free


@pytest.mark.gpu
def test_damage_anywhere_in_a_long_step_is_found(pcl, torch, ctx):
    # more pages than the threads look at in one round, one of them outside the
    # pools
    batch = DeviceBatch(pcl, torch, 3, 6000, 1, 12000, 11000)
    ctx.page_reset(batch.desc)
    good = batch.a["free_pages"].clone()
    for u in (0, 255, 4095, 4096, 8191, 10500, 10999):
        batch.a["free_pages"][12000 - 1 - u] = 12000
        ctx.page_step(batch.desc, batch.put([5000, 1000, 5000]))
        assert ctx.sync() == BAD_PAGES
        state = batch.state()
        assert state["counters"].tolist() == [12000, 11000, 11000, 0]
        assert np.flatnonzero(state["slots"] == -1).tolist() == [u]
        assert np.count_nonzero(state["table"] == -1) == 3 * 6000 - 11000 + 1
        batch.a["free_pages"].copy_(good)
    batch.a["free_pages"][12000 - 1 - 11000] = 12000  # (the next page is not taken)
    ctx.page_step(batch.desc, batch.put([5000, 1000, 5000]))
    assert ctx.sync() == 0 and batch.state()["counters"][3] == 1


@pytest.mark.gpu
def test_released_pages_past_32_bits_are_refused(pcl, torch, ctx):
    # lengths that add up to 2^32 pages, of pools of 2^21
    n = 1 << 21
    batch = DeviceBatch(pcl, torch, 2048, n, 1, n, 64)
    ctx.page_reset(batch.desc)
    batch.a["lengths"].fill_(n)
    ctx.page_release(batch.desc, batch.put([1] * 2048))
    assert ctx.sync() == BAD_PAGES
    assert bool((batch.a["lengths"] == n).all()) and int(batch.a["counters"][0]) == n
    # or that many stay
    batch.a["counters"][0] = 0
    ctx.page_release(batch.desc, batch.put([1] + [0] * 2047))
    assert ctx.sync() == BAD_PAGES
    assert bool((batch.a["lengths"] == n).all()) and int(batch.a["counters"][0]) == 0
    del batch
    torch.cuda.empty_cache()


def dtype_of(torch, name):
    return torch.float32 if name == "f32" else torch.bfloat16


class Pools:
    """One layer's pages, every value a NaN until it is written."""

    def __init__(self, pcl, torch, pages, page, kvheads, dim, dtype):
        self.k = torch.full((pages, page, kvheads, dim), float("nan"), device="cuda:0",
                            dtype=dtype_of(torch, dtype))
        self.v = self.k.clone()
        self.desc = pcl.page_pools(
            k=self.k.data_ptr(), v=self.v.data_ptr(),
            type=pcl.CACHE_F32 if dtype == "f32" else pcl.CACHE_BF16, pages=pages,
            page_tokens=page, kvheads=kvheads, dim=dim)

    def rows(self, slots):
        """(K, V) rows of the slots, widened."""
        return [x.view(-1, *x.shape[2:])[slots].float() for x in (self.k, self.v)]


def bits(x):
    return x.contiguous().view(x.new_empty(0, dtype=x.dtype).dtype).cpu().float().numpy() \
        .view(np.uint32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(2, 16), (1, 48), (8, 256), (3, 512), (40, 64)],
                         ids=lambda h: "%dx%d" % h)
@pytest.mark.parametrize("n", [1, 5, 130])
def test_append_moves_rows_to_their_slots(pcl, torch, ctx, dtype, heads, n):
    kvheads, dim = heads
    page, pages = 7, 40
    pools = Pools(pcl, torch, pages, page, kvheads, dim, dtype)
    g = torch.Generator(device="cuda:0")
    g.manual_seed(n + dim)
    keys = torch.randn((n, kvheads, dim), generator=g, device="cuda:0")
    values = torch.randn((n, kvheads, dim), generator=g, device="cuda:0")
    # values at the ends of the range and a NaN keep their place too
    keys[0, 0, :4] = torch.tensor([float("inf"), -0.0, 1e-45, float("nan")])
    slots = torch.randperm(pages * page, generator=g, device="cuda:0")[:n].int()
    if n > 1:
        slots[n // 2] = -1
    ctx.paged_append(pools.desc, slots.data_ptr(), keys.data_ptr(), values.data_ptr(), n)
    assert ctx.sync() == 0
    want = [torch.full_like(pools.k, float("nan")) for _ in range(2)]
    for out, src in zip(want, (keys, values)):
        live = slots >= 0
        out.view(-1, kvheads, dim)[slots[live].long()] = src[live].to(out.dtype)
    for got, out in zip((pools.k, pools.v), want):
        assert torch.equal(torch.isnan(got), torch.isnan(out))
        keep = ~torch.isnan(out)
        assert np.array_equal(bits(got[keep]), bits(out[keep]))


@pytest.mark.gpu
def test_append_reports_slots_past_the_pools(pcl, torch, ctx):
    pools = Pools(pcl, torch, 3, 5, 2, 64, "f32")
    rows = torch.randn((3, 2, 64), device="cuda:0")
    for bad in (15, 1 << 30, (1 << 31) - 1):
        slots = torch.tensor([2, bad, 9], dtype=torch.int32, device="cuda:0")
        pools.k.fill_(7.0)
        ctx.paged_append(pools.desc, slots.data_ptr(), rows.data_ptr(), rows.data_ptr(), 3)
        assert ctx.sync() == BAD_PAGES
        flat = pools.k.view(15, 2, 64)
        assert torch.equal(flat[2], rows[0]) and torch.equal(flat[9], rows[2])
        assert int((flat == 7.0).all(-1).all(-1).sum()) == 13


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(2, 1, 16), (4, 2, 32), (6, 3, 64), (8, 8, 128), (16, 8, 256),
                                   (16, 2, 512)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("n,own_v", [(1, True), (9, False), (70, True)])
def test_transformed_append_equals_single_tokens(pcl, torch, ctx, dtype, heads, n, own_v):
    qheads, kvheads, dim = heads
    g = torch.Generator(device="cuda:0")
    g.manual_seed(dim + n)

    def randn(*s):
        return torch.randn(s, generator=g, device="cuda:0")

    scales = [1.0 + 0.2 * np.random.default_rng(s).standard_normal(dim) for s in (1, 2)]
    tr = pcl.HeadTransform(ctx, qheads, kvheads, dim, *scales, 1e-6, 10000.0)
    limit, page, pages = 3000, 16, 9
    pools = Pools(pcl, torch, pages, page, kvheads, dim, dtype)
    q, k, v = randn(n, qheads, dim), randn(n, kvheads, dim), randn(n, kvheads, dim)
    slots = torch.randperm(pages * page, generator=g, device="cuda:0")[:n].int()
    positions = torch.randint(0, limit, (n,), generator=g, device="cuda:0", dtype=torch.int32)
    positions[0] = limit - 1
    positions[-1] = 0 if n > 1 else limit - 1
    if n > 4:
        slots[3], positions[3] = -1, -5  # left out
        k[3] = float("nan")
    q_out = torch.full_like(q, 3.5)
    tr.append_paged(pools.desc, slots.data_ptr(), positions.data_ptr(), limit, q.data_ptr(),
                    k.data_ptr(), v.data_ptr() if own_v else None, n, q_out.data_ptr())
    assert ctx.sync() == 0
    written = [torch.full_like(pools.k, float("nan")) for _ in range(2)]
    for i in range(n):
        if int(slots[i]) < 0:
            assert bool((q_out[i] == 3.5).all())
            continue
        one = [torch.empty_like(x[:1]) for x in (q, k, v)]
        tr.prepare(q[i].data_ptr(), k[i].data_ptr(), v[i].data_ptr() if own_v else None, 1,
                   int(positions[i]), *[x.data_ptr() for x in one])
        assert np.array_equal(bits(q_out[i]), bits(one[0][0]))
        for out, x in zip(written, one[1:]):
            out.view(-1, kvheads, dim)[int(slots[i])] = x[0].to(out.dtype)
    assert ctx.sync() == 0
    for got, want in zip((pools.k, pools.v), written):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        keep = ~torch.isnan(want)
        assert np.array_equal(bits(got[keep]), bits(want[keep]))
    tr.close()


@pytest.mark.gpu
def test_transformed_append_refusals(pcl, torch, ctx):
    tr = pcl.HeadTransform(ctx, 4, 2, 64, np.ones(64), np.ones(64), 1e-6, 10000.0, sliding=True)
    pools = Pools(pcl, torch, 3, 5, 2, 64, "f32")
    q, k = torch.randn((2, 4, 64), device="cuda:0"), torch.randn((2, 2, 64), device="cuda:0")
    slots = torch.tensor([1, 4], dtype=torch.int32, device="cuda:0")
    positions = torch.tensor([2, 7], dtype=torch.int32, device="cuda:0")
    out = torch.empty_like(q)

    def call(desc=pools.desc, limit=8, v=k.data_ptr(), n=2, q_ptr=q.data_ptr()):
        tr.append_paged(desc, slots.data_ptr(), positions.data_ptr(), limit, q_ptr, k.data_ptr(),
                        v, n, out.data_ptr())

    for kw, kind in ((dict(limit=0), "ResourceLimit"), (dict(limit=(1 << 24) + 1), "ResourceLimit"),
                     (dict(v=None), "InvalidShape"), (dict(n=-1), "InvalidShape"),
                     (dict(q_ptr=q.data_ptr() + 4), "InvalidShape"),
                     (dict(desc=pcl.page_pools(k=64, v=64, pages=3, page_tokens=5, kvheads=1,
                                               dim=64)), "InvalidShape"),
                     (dict(desc=pcl.page_pools(k=64, v=64, pages=3, page_tokens=5, kvheads=2,
                                               dim=128)), "InvalidShape")):
        with pytest.raises(pcl.AttentionError) as e:
            call(**kw)
        assert e.value.kind == kind
    call(n=0)
    assert ctx.sync() == 0
    # positions and slots out of range leave the row out, with the error
    for name, bad in (("positions", 8), ("positions", -1), ("slots", 15), ("slots", 1 << 30)):
        keep = {"positions": positions, "slots": slots}[name]
        old = keep.clone()
        keep[1] = bad
        out.fill_(2.5)
        call()
        assert ctx.sync() == BAD_PAGES
        assert bool((out[1] == 2.5).all()) and not bool((out[0] == 2.5).any())
        keep.copy_(old)
    call()
    assert ctx.sync() == 0
    tr.close()


class Cache:
    """Requests of the given lengths over pages in a random order, filled with
    keys and values; the pages' other slots hold NaNs."""

    def __init__(self, pcl, torch, heads, lengths, page, dtype, seed, scale=1.0):
        self.pcl, self.torch, self.heads = pcl, torch, heads
        _, kvheads, dim = heads
        rng = np.random.default_rng(seed)
        held = [-(-n // page) for n in lengths]
        pages = sum(held) + 3
        order = rng.permutation(pages)
        self.stride = max(held + [1]) + 2
        table = np.full((len(lengths), self.stride), -1, np.int32)
        self.pools = Pools(pcl, torch, pages, page, kvheads, dim, dtype)
        g = torch.Generator(device="cuda:0")
        g.manual_seed(seed)
        self.k, self.v = [], []  # each request's rows, as the pages hold them
        at = 0
        for b, (n, h) in enumerate(zip(lengths, held)):
            table[b, :h] = order[at:at + h]
            at += h
            position = np.arange(n)
            slots = torch.from_numpy(table[b, position // page].astype(np.int64) * page +
                                     position % page).to("cuda:0")
            for keep, pool in ((self.k, self.pools.k), (self.v, self.pools.v)):
                rows = torch.randn((n, kvheads, dim), generator=g, device="cuda:0") * scale
                rows = rows.to(pool.dtype)
                pool.view(-1, kvheads, dim)[slots] = rows
                keep.append(rows.float())
        self.lengths = list(lengths)
        self.page = page
        self.table = torch.from_numpy(table).to("cuda:0")
        self.dlengths = torch.tensor(lengths, dtype=torch.int32, device="cuda:0")

    def attend(self, ctx, q, rows=None, window=0, max_length=None, softcap=0.0, q_scale=None,
               out=None, **kw):
        qheads, _, dim = self.heads
        torch = self.torch
        out = torch.full_like(q, 9.5) if out is None else out
        drows = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda:0")
        d = ctx.paged_desc(
            pools=self.pools.desc, q=q.data_ptr(), q_stride=q.stride(0), q_rows=q.shape[0],
            qheads=qheads, table=self.table.data_ptr(), table_stride=self.stride,
            lengths=self.dlengths.data_ptr(), rows=drows.data_ptr() if rows is not None else None,
            requests=len(self.lengths), max_length=max_length or self.stride * self.page,
            window=window, q_scale=scale_of(dim) if q_scale is None else q_scale, softcap=softcap,
            out=out.data_ptr(), o_stride=out.stride(0))
        for n, v in kw.items():
            setattr(d, n, v)
        # the context may be on another stream than the tensors
        torch.cuda.synchronize()
        ctx.paged_attention(d)
        torch.cuda.synchronize()
        return out

    def contiguous(self, ctx, q, b, window=0, softcap=0.0, kernel=0):
        """The same request through pcl_attention_launch."""
        qheads, kvheads, dim = self.heads
        out = self.torch.empty((1, qheads * dim), device="cuda:0")
        q = q[:, :qheads * dim].contiguous()
        n = self.lengths[b]
        k, v = self.k[b].contiguous(), self.v[b].contiguous()
        self.torch.cuda.synchronize()
        ctx.launch(ctx.desc(
            q=q.data_ptr(), q_stride=qheads * dim, nq=1, k0=k.data_ptr(), v0=v.data_ptr(), n0=n,
            qheads=qheads, kvheads=kvheads, dim=dim, kh_first=0, kh_end=kvheads, causal=1,
            window=window, first_query=n - 1, q_scale=scale_of(dim), softcap=softcap,
            out=out.data_ptr(), o_stride=qheads * dim, kernel=kernel))
        self.torch.cuda.synchronize()
        return out[0]

    def plain(self, q, b, window=0, softcap=0.0):
        """A softmax in 64 bits."""
        torch = self.torch
        qheads, kvheads, dim = self.heads
        lo = max(0, self.lengths[b] - window) if window else 0
        k, v = self.k[b][lo:].double(), self.v[b][lo:].double()
        # the engine scales the query in f32
        x = (q[:qheads * dim] * np.float32(scale_of(dim))).double().view(kvheads, -1, dim)
        s = torch.matmul(x, k.permute(1, 2, 0).contiguous())
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        w = torch.softmax(s, -1)
        return torch.matmul(w, v.permute(1, 0, 2).contiguous()).reshape(-1)


def scale_of(dim):
    return float(np.float32(1.0 / np.sqrt(dim)))


def tolerance(keys, dim):
    """Bound of |out - exact| over the size of the values (at most ~5 for a few
    million normals): scores of |s| <= sqrt(dim) * 5 * 5 / sqrt(dim) = 25 with
    dim fmas each of half a step (2^-24 of the partial sums, at most dim * 25 *
    2^-24) are off by dim * 25 * 2^-24, and so, as a factor, is each weight; the
    sums over the keys add keys * 2^-24 and the exponentials 2 steps."""
    return 5 * (2 * dim * 25 + 2 * keys + 64) * 2.0 ** -24


HEADS = [(16, 8, 256), (16, 2, 512), (32, 8, 128), (16, 4, 64), (10, 2, 80), (3, 3, 16),
         (20, 1, 48), (2, 1, 272), (33, 1, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("window", [0, 100])
def test_attention_has_the_contiguous_bits(pcl, torch, ctx, dtype, heads, window):
    # lengths of one token, around tiles, pages and chunks, of several chunks
    # and of more than one span
    lengths = [1, 2, 15, 16, 17, 33, 255, 256, 257, 300, 511, 513, 1025, 4097, 5000]
    page = {256: 16, 512: 7, 128: 48, 64: 300}.get(heads[2], 5)
    cache = Cache(pcl, torch, heads, lengths, page, dtype, heads[2] + window)
    q = torch.randn((len(lengths), heads[0] * heads[2]), device="cuda:0")
    out = cache.attend(ctx, q, window=window)
    assert ctx.sync() == 0
    for b, n in enumerate(lengths):
        want = cache.contiguous(ctx, q[b:b + 1], b, window)
        # adding 0 makes a negative zero positive
        assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0)), n
        exact = cache.plain(q[b], b, window)
        assert float((out[b].double() - exact).abs().max()) <= tolerance(n, heads[2]), n
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(4, 4, 64), (16, 2, 64), (12, 1, 64), (8, 4, 128), (5, 1, 128),
                                   (16, 8, 256), (14, 2, 256), (4, 2, 512), (16, 2, 512),
                                   (16, 1, 512), (2, 1, 496)],
                         ids=lambda h: "x".join(map(str, h)))
def test_launches_of_few_items(pcl, torch, ctx, dtype, heads):
    # every item with a CU to itself: the kernels with two buffers a wave
    for lengths in ([1], [100], [257, 40], [64, 2, 700]):
        cache = Cache(pcl, torch, heads, lengths, 16, dtype, sum(lengths))
        q = torch.randn((len(lengths), heads[0] * heads[2]), device="cuda:0")
        out = cache.attend(ctx, q, max_length=max(lengths))
        loose = cache.attend(ctx, q)
        assert ctx.sync() == 0
        for b, n in enumerate(lengths):
            want = cache.contiguous(ctx, q[b:b + 1], b)
            assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0)), (lengths, b)
            assert np.array_equal(bits(loose[b]), bits(out[b]))
            exact = cache.plain(q[b], b)
            assert float((out[b].double() - exact).abs().max()) <= tolerance(n, heads[2])
        assert ctx.sync() == 0


@pytest.mark.gpu
def test_uniform_batches_of_whole_chunks(pcl, torch, ctx):
    # more items than workgroups: each takes several, full chunks throughout
    for heads, dtype in (((16, 8, 256), "bf16"), ((16, 2, 512), "f32"), ((4, 4, 64), "bf16")):
        cache = Cache(pcl, torch, heads, [2048] * 24, 64, dtype, 77)
        q = torch.randn((24, heads[0] * heads[2]), device="cuda:0")
        first = cache.attend(ctx, q)
        again = cache.attend(ctx, q)
        assert ctx.sync() == 0
        assert np.array_equal(bits(first), bits(again))
        for b in (0, 11, 23):
            want = cache.contiguous(ctx, q[b:b + 1], b)
            assert np.array_equal(bits(first[b] + 0.0), bits(want + 0.0))
        assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(16, 8, 256), (16, 2, 512)], ids=["d256", "d512"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_requests(pcl, torch, ctx, heads, dtype):
    # several spans; one request alone and among others has the same bits
    lengths = [20000, 3, 70001, 9000]
    cache = Cache(pcl, torch, heads, lengths, 64, dtype, 11)
    q = torch.randn((4, heads[0] * heads[2]), device="cuda:0")
    out = cache.attend(ctx, q)
    for b, n in enumerate(lengths):
        want = cache.contiguous(ctx, q[b:b + 1], b)
        assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0)), n
        alone = cache.attend(ctx, q, rows=[i if i == b else -1 for i in range(4)])
        assert np.array_equal(bits(alone[b]), bits(out[b]))
        exact = cache.plain(q[b], b)
        assert float((out[b].double() - exact).abs().max()) <= tolerance(n, heads[2]), n
    windowed = cache.attend(ctx, q, window=6000)
    for b, n in enumerate(lengths):
        want = cache.contiguous(ctx, q[b:b + 1], b, 6000)
        assert np.array_equal(bits(windowed[b] + 0.0), bits(want + 0.0)), n
    assert ctx.sync() == 0


@pytest.mark.gpu
def test_a_window_without_a_limit(pcl, torch):
    # windows up to the last int64_t attend every key, through a workspace of
    # that launch alone
    heads = (4, 2, 64)
    cache = Cache(pcl, torch, heads, [700, 40, 3000], 16, "f32", 41)
    q = torch.randn((3, 256), device="cuda:0")
    for window in (3000, 1 << 40, (1 << 63) - 1):
        torch.cuda.synchronize()
        own = pcl.Context(0)
        out = cache.attend(own, q, window=window)
        for b in range(3):
            want = cache.contiguous(own, q[b:b + 1], b)
            assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0))
        assert own.sync() == 0
        own.close()


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.75, 50.0])
def test_softcap(pcl, torch, ctx, softcap):
    for heads, dtype in (((16, 8, 256), "f32"), ((32, 8, 128), "bf16"), ((10, 2, 80), "f32")):
        cache = Cache(pcl, torch, heads, [1, 300, 700], 16, dtype, 3)
        q = 6 * torch.randn((3, heads[0] * heads[2]), device="cuda:0")
        out = cache.attend(ctx, q, softcap=softcap)
        for b in range(3):
            want = cache.contiguous(ctx, q[b:b + 1], b, softcap=softcap)
            assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0))
    assert ctx.sync() == 0


def exact_and_bound(cache, q, b, window=0, softcap=0.0):
    """The attention of request b in 64 bits, and a bound of the kernels' error for
    each value, from the request's own numbers. With u = 2^-24, half an f32 step:

    a score is a chain of dim fmas from zero, off by at most 1.01 dim u sum|q_d k_d|
    (1.01 for the higher powers of u; the scaled query is the kernels' own); a cap
    passes that on at most as it is and adds 20 u of its value (exp off by 13 u at
    worst where 1 - exp(-2 |t|) cancels, and the roundings of t, the sums, the
    reciprocal and the product).
    exp(x) is exp2 of x log2(e), x a difference: 3 |x| u of the argument and 2 u of
    the instruction. A term is multiplied by the exp of its own tile and by the
    factors of the tiles, chunks and spans behind it, whose arguments are the steps
    of one running maximum: together at most R = max s - s_t, with 2 u each.
    A term passes through at most 256 fmas and 8 factors of its chunk and one fma
    per chunk of its span and per span, two more where a part enters a merge.
    The numerator's terms are thus off by e (relative), the denominator's by no
    more, and their quotient by 2.02 e of the sum of |w v|, and 4 u of itself."""
    torch = cache.torch
    qheads, kvheads, dim = cache.heads
    n = cache.lengths[b]
    lo = max(0, n - window) if window else 0
    k, v = cache.k[b][lo:].double(), cache.v[b][lo:].double()
    x = (q[:qheads * dim] * np.float32(scale_of(dim))).double().view(kvheads, -1, dim)
    kt = k.permute(1, 2, 0).contiguous()
    s, size = torch.matmul(x, kt), torch.matmul(x.abs(), kt.abs())
    capped = softcap * torch.tanh(s / softcap) if softcap else s
    w = torch.softmax(capped, -1)
    vt = v.permute(1, 0, 2).contiguous()
    exact = torch.matmul(w, vt)
    spans = n // (16 * 256) + 1
    e = 1.01 * dim * size.amax(-1, keepdim=True) + \
        (20 * capped.abs().amax(-1, keepdim=True) if softcap else 0) + \
        3 * (capped.amax(-1, keepdim=True) - capped.amin(-1, keepdim=True)) + \
        2 * (1 + 8 + 17 + spans + 1) + 256 + 8 + 16 + spans + 2
    u = 2.0 ** -24
    bound = 2.02 * e * u * torch.matmul(w, vt.abs()) + 4 * u * exact.abs()
    return exact.reshape(-1), bound.reshape(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(16, 8, 256), (16, 2, 512), (32, 8, 128), (4, 4, 64)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 6000])
def test_long_requests_in_64_bits(pcl, torch, ctx, heads, dtype, window):
    # a bound well below the outputs, which shrink with the number of keys
    lengths = [20000, 3, 70001, 257]
    cache = Cache(pcl, torch, heads, lengths, 64, dtype, 13)
    q = torch.randn((4, heads[0] * heads[2]), device="cuda:0")
    out = cache.attend(ctx, q, window=window)
    assert ctx.sync() == 0
    for b, n in enumerate(lengths):
        exact, bound = exact_and_bound(cache, q[b], b, window)
        assert float(bound.max()) < 0.5 * float(exact.abs().mean()), n
        assert bool(((out[b].double() - exact).abs() <= bound).all()), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("softcap", [0.75, 3.0, 50.0])
def test_softcap_in_64_bits(pcl, torch, ctx, dtype, softcap):
    # scores far past the cap, around it and far below it
    for heads in ((16, 8, 256), (32, 8, 128), (10, 2, 80)):
        cache = Cache(pcl, torch, heads, [1, 300, 700, 5000], 16, dtype, 3)
        q = 6 * torch.randn((4, heads[0] * heads[2]), device="cuda:0")
        out = cache.attend(ctx, q, softcap=softcap)
        assert ctx.sync() == 0
        for b in range(4):
            exact, bound = exact_and_bound(cache, q[b], b, softcap=softcap)
            # and the cap shows
            other = exact_and_bound(cache, q[b], b)[0] if b else -exact
            assert float(bound.max()) < 0.5 * float((exact - other).abs().mean())
            assert bool(((out[b].double() - exact).abs() <= bound).all()), (heads, b)


@pytest.mark.gpu
def test_rows_strides_and_requests_left_out(pcl, torch, ctx):
    # requests without a row or keys, rows in another order, padded strides:
    # what no request owns stays as it was
    heads = (4, 2, 64)
    lengths = [40, 0, 300, 7, 600, 1]
    rows = [5, 2, -1, 0, 3, -7]
    cache = Cache(pcl, torch, heads, lengths, 16, "f32", 5)
    q = torch.randn((8, 4 * 64 + 12), device="cuda:0")
    q[[1, 2, 4, 6, 7]] = float("nan")  # rows of no active request are not read
    out = torch.full((8, 4 * 64 + 8), 9.5, device="cuda:0")
    cache.attend(ctx, q, rows=rows, out=out)
    assert ctx.sync() == 0
    assert bool((out[:, 256:] == 9.5).all())
    for b, r in enumerate(rows):
        if r < 0 or lengths[b] == 0:
            continue
        want = cache.contiguous(ctx, q[r:r + 1], b)
        assert np.array_equal(bits(out[r, :256] + 0.0), bits(want + 0.0))
    assert bool((out[[1, 2, 4, 6, 7]] == 9.5).all())
    # nobody: nothing happens
    out.fill_(9.5)
    cache.attend(ctx, q, rows=[-1] * 6, out=out)
    cache.attend(ctx, q, rows=rows, out=out, requests=0)
    assert ctx.sync() == 0
    assert bool((out == 9.5).all())


@pytest.mark.gpu
def test_device_side_errors(pcl, torch, ctx):
    heads = (4, 2, 64)
    cache = Cache(pcl, torch, heads, [40, 300, 700], 16, "f32", 6)
    q = torch.randn((3, 256), device="cuda:0")
    good = cache.attend(ctx, q)
    assert ctx.sync() == 0

    def others(out, b):
        assert all(torch.equal(out[i], good[i]) for i in range(3) if i != b)

    # a row past q_rows and a length past max_length or below zero
    for rows, want in (([0, 3, 2], BAD_PAGES), ([0, 1 << 30, 2], BAD_PAGES), ([0, -1, 2], 0)):
        out = cache.attend(ctx, q, rows=rows)
        assert ctx.sync() == want
        others(out, 1)
        assert bool((out[1] == 9.5).all())
    for n, want in ((-3, 0), (1 << 30, BAD_PAGES), (401, BAD_PAGES)):
        cache.dlengths[1] = n
        out = cache.attend(ctx, q, max_length=None if n != 401 else 400, rows=[0, 1, -1])
        assert ctx.sync() == want
        assert torch.equal(out[0], good[0]) and bool((out[1:] == 9.5).all())
    cache.dlengths[1] = 300
    # pages outside the pools are reported and read as page 0
    keep = cache.table.clone()
    pages = cache.pools.k.shape[0]
    cache.pools.k[0] = 1.0
    cache.pools.v[0] = 1.0
    good = cache.attend(ctx, q)
    assert ctx.sync() == 0
    for bad in (pages, -1, (1 << 31) - 1, -(1 << 31)):
        cache.table[1, 3] = bad
        out = cache.attend(ctx, q)
        assert ctx.sync() == BAD_PAGES
        others(out, 1)
        cache.table.copy_(keep)
    # a NaN in an attended key or value is reported, one outside is not read
    slot = int(cache.table[2, 0]) * 16 + 3
    flat_k, flat_v = (x.view(-1, 2, 64) for x in (cache.pools.k, cache.pools.v))
    for flat, bit in ((flat_k, 1), (flat_v, 2)):
        old = flat[slot].clone()
        flat[slot, 1, 5] = float("nan")
        cache.attend(ctx, q)
        assert ctx.sync() & bit
        inside = cache.attend(ctx, q, window=600)
        assert ctx.sync() == 0 and bool(torch.isfinite(inside).all())
        flat[slot] = old


@pytest.mark.gpu
def test_shared_pages(pcl, torch, ctx):
    # two requests over the same first pages: a common prompt
    heads = (8, 2, 128)
    cache = Cache(pcl, torch, heads, [512, 600], 32, "bf16", 8)
    cache.table[1, :16] = cache.table[0, :16]
    for keep in (cache.k, cache.v):
        keep[1][:512] = keep[0]
    q = torch.randn((2, 8 * 128), device="cuda:0")
    out = cache.attend(ctx, q)
    for b in range(2):
        want = cache.contiguous(ctx, q[b:b + 1], b)
        assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0))
    assert ctx.sync() == 0


@pytest.mark.gpu
def test_slots_past_32_bit_offsets(pcl, torch, ctx):
    # pools of more than 2^32 bytes (and 2^31 values): rows behind that mark
    kvheads, dim, page = 8, 256, 64
    pages = (1 << 31) // (page * kvheads * dim) + 40
    k = torch.empty((pages, page, kvheads, dim), device="cuda:0", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    pools = pcl.page_pools(k=k.data_ptr(), v=v.data_ptr(), type=pcl.CACHE_BF16, pages=pages,
                           page_tokens=page, kvheads=kvheads, dim=dim)
    n = 300
    table = torch.tensor([[pages - 1, 2, pages - 3, pages - 2, pages - 7]], dtype=torch.int32,
                         device="cuda:0")
    position = torch.arange(n, device="cuda:0")
    slots = (table[0, position // page] * page + position % page).int()
    keys = torch.randn((n, kvheads, dim), device="cuda:0").bfloat16().float()
    values = torch.randn((n, kvheads, dim), device="cuda:0").bfloat16().float()
    ctx.paged_append(pools, slots.data_ptr(), keys.data_ptr(), values.data_ptr(), n)
    assert ctx.sync() == 0
    assert torch.equal(k.view(-1, kvheads, dim)[slots.long()].float(), keys)
    q = torch.randn((1, 16 * dim), device="cuda:0")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda:0")
    outs = [torch.empty_like(q) for _ in range(2)]
    ctx.paged_attention(ctx.paged_desc(
        pools=pools, q=q.data_ptr(), q_stride=16 * dim, q_rows=1, qheads=16,
        table=table.data_ptr(), table_stride=5, lengths=lengths.data_ptr(), requests=1,
        max_length=320, out=outs[0].data_ptr(), o_stride=16 * dim, q_scale=scale_of(dim)))
    ctx.launch(ctx.desc(
        q=q.data_ptr(), q_stride=16 * dim, nq=1, k0=keys.data_ptr(), v0=values.data_ptr(), n0=n,
        qheads=16, kvheads=8, dim=dim, kh_first=0, kh_end=8, causal=1, first_query=n - 1,
        q_scale=scale_of(dim), out=outs[1].data_ptr(), o_stride=16 * dim))
    assert ctx.sync() == 0
    assert np.array_equal(bits(outs[0] + 0.0), bits(outs[1] + 0.0))


@pytest.mark.gpu
def test_many_requests(pcl, torch, ctx):
    # as many requests as a batch may have, most of a single chunk
    rng = np.random.default_rng(4)
    lengths = [int(n) for n in rng.integers(0, 40, 2048)]
    lengths[7], lengths[2047], lengths[1000] = 600, 258, 1025
    heads = (2, 1, 64)
    cache = Cache(pcl, torch, heads, lengths, 16, "f32", 12)
    q = torch.randn((2048, 128), device="cuda:0")
    out = cache.attend(ctx, q)
    assert ctx.sync() == 0
    for b in [0, 1, 7, 500, 999, 1000, 1001, 2046, 2047] + list(range(40, 80)):
        if lengths[b] == 0:
            assert bool((out[b] == 9.5).all())
            continue
        want = cache.contiguous(ctx, q[b:b + 1], b)
        assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0)), b


@pytest.mark.gpu
def test_timing_counts_the_launches(pcl, torch):
    own = pcl.Context(0)
    cache = Cache(pcl, torch, (4, 2, 64), [700, 40], 16, "f32", 22)
    q = torch.randn((2, 256), device="cuda:0")
    cache.attend(own, q)
    own.set_timing(True)
    cache.attend(own, q)
    cache.attend(own, q, rows=[-1, 1], max_length=40)  # (one chunk at most: no combine)
    assert own.sync() == 0  # (the longer request has no row)
    ms, launches = own.timing()
    assert launches == (2, 1) and ms[0] > 0 and ms[1] > 0
    own.set_timing(False)
    cache.attend(own, q)
    assert own.timing()[1] == (0, 0)
    own.close()


@pytest.mark.gpu
def test_another_stream(pcl, torch):
    # a context that owns its stream; inputs handed over by an event
    heads = (16, 8, 256)
    cache = Cache(pcl, torch, heads, [700, 40], 16, "f32", 21)
    q = torch.randn((2, 16 * 256), device="cuda:0")
    torch.cuda.synchronize()
    own = pcl.Context(0)
    out = torch.full_like(q, 9.5)
    torch.cuda.synchronize()
    cache.attend(own, q, out=out)
    assert own.sync() == 0
    for b in range(2):
        want = cache.contiguous(own, q[b:b + 1], b)
        assert own.sync() == 0
        assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0))
    own.close()


@pytest.mark.gpu
def test_two_contexts_at_once(pcl, torch):
    # each has its stream, workspace and error flag; the pages are shared
    heads = (16, 8, 256)
    cache = Cache(pcl, torch, heads, [3000] * 12, 16, "bf16", 23)
    q = [torch.randn((12, 16 * 256), device="cuda:0") for _ in range(2)]
    out = [torch.zeros_like(x) for x in q]
    own = [pcl.Context(0) for _ in q]
    descs = [c.paged_desc(
        pools=cache.pools.desc, q=x.data_ptr(), q_stride=16 * 256, q_rows=12, qheads=16,
        table=cache.table.data_ptr(), table_stride=cache.stride,
        lengths=cache.dlengths.data_ptr(), requests=12, max_length=3000, q_scale=scale_of(256),
        out=o.data_ptr(), o_stride=16 * 256) for c, x, o in zip(own, q, out)]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, d in zip(own, descs):
            c.paged_attention(d)
    assert [c.sync() for c in own] == [0, 0]
    for c, x, o in zip(own, q, out):
        for b in (0, 5, 11):
            want = cache.contiguous(c, x[b:b + 1], b)
            assert c.sync() == 0
            assert np.array_equal(bits(o[b] + 0.0), bits(want + 0.0))
        c.close()


# ---- a run of them together -------------------------------------------------

class Server:
    """One layer of a batched decoder: the step's raw projections through the
    head transform into the pages, attention, and the output block."""

    def __init__(self, pcl, torch, ctx, heads, requests, page, pages, stride, rows, window, dtype):
        qheads, kvheads, dim = heads
        self.pcl, self.torch, self.ctx, self.heads = pcl, torch, ctx, heads
        self.batch = DeviceBatch(pcl, torch, requests, stride, page, pages, rows)
        self.pools = Pools(pcl, torch, pages, page, kvheads, dim, dtype)
        self.limit = stride * page
        scale = 1.0 + 0.1 * np.random.default_rng(0).standard_normal(dim)
        self.transform = pcl.HeadTransform(ctx, qheads, kvheads, dim, scale, scale[::-1], 1e-6,
                                           10000.0)
        dev = {"device": "cuda:0"}
        self.raw = [torch.zeros((rows, h, dim), **dev) for h in (qheads, kvheads, kvheads)]
        self.q = torch.zeros((rows, qheads * dim), **dev)
        self.attended = torch.zeros((rows, qheads * dim), **dev)
        hidden = 96
        g = torch.Generator(device="cuda:0")
        g.manual_seed(1)
        self.w = torch.randn((hidden, qheads * dim), generator=g, **dev)
        self.post = torch.ones(hidden, **dev)
        self.residual = torch.ones((rows, hidden), **dev)
        self.projected, self.result = (torch.zeros((rows, hidden), **dev) for _ in range(2))
        a = self.batch.a
        self.desc = ctx.paged_desc(
            pools=self.pools.desc, q=self.q.data_ptr(), q_stride=qheads * dim, q_rows=rows,
            qheads=qheads, table=a["table"].data_ptr(), table_stride=stride,
            lengths=a["step_lengths"].data_ptr(), rows=a["newest"].data_ptr(), requests=requests,
            max_length=self.limit, window=window, q_scale=scale_of(dim),
            out=self.attended.data_ptr(), o_stride=qheads * dim)
        self.rows, self.window, self.hidden = rows, window, hidden
        ctx.reserve(ctx.paged_workspace_bytes(self.desc))
        ctx.page_reset(self.batch.desc)

    def step(self, commit=True):
        a, ctx = self.batch.a, self.ctx
        ctx.page_step(self.batch.desc, self.batch.words.data_ptr())
        self.transform.append_paged(self.pools.desc, a["slots"].data_ptr(),
                                    a["positions"].data_ptr(), self.limit,
                                    *[x.data_ptr() for x in self.raw], self.rows,
                                    self.q.data_ptr())
        ctx.paged_attention(self.desc)
        ctx.attention_output(self.attended.data_ptr(), self.rows, self.attended.shape[1],
                             self.w.data_ptr(), self.hidden, self.post.data_ptr(), 1e-6,
                             self.residual.data_ptr(), self.projected.data_ptr(),
                             self.result.data_ptr())
        if commit:
            ctx.page_commit(self.batch.desc)


class Reference:
    """The same requests one by one through the layer cache of one sequence."""

    def __init__(self, server):
        self.s = server
        self.raw = {}  # request -> list of (q, k, v) rows

    def take(self, model):
        """The step's rows, as the model lays them out."""
        for t, b in enumerate(model.row_request):
            self.raw.setdefault(b, [])
            del self.raw[b][model.positions[t]:]
            self.raw[b].append([x[t].clone() for x in self.s.raw])

    def keep(self, lengths):
        for b, rows in self.raw.items():
            del rows[lengths[b]:]

    def attended(self, b):
        """The newest token of request b over its rows so far."""
        s, torch = self.s, self.s.torch
        qheads, kvheads, dim = s.heads
        rows = self.raw[b]
        n = len(rows)
        raw = [torch.stack([r[i] for r in rows]) for i in range(3)]
        q, k, v = (torch.empty_like(x) for x in raw)
        torch.cuda.synchronize()  # the context is on another stream
        s.transform.prepare(*[x.data_ptr() for x in raw], n, 0, *[x.data_ptr() for x in (q, k, v)])
        torch.cuda.synchronize()
        if s.pools.k.dtype == torch.bfloat16:
            k, v = k.bfloat16().float(), v.bfloat16().float()
        out = torch.empty((1, qheads * dim), device="cuda:0")
        torch.cuda.synchronize()
        s.ctx.launch(s.ctx.desc(
            q=q[n - 1].data_ptr(), q_stride=qheads * dim, nq=1, k0=k.data_ptr(), v0=v.data_ptr(),
            n0=n, qheads=qheads, kvheads=kvheads, dim=dim, kh_first=0, kh_end=kvheads, causal=1,
            window=s.window, first_query=n - 1, q_scale=scale_of(dim), out=out.data_ptr(),
            o_stride=qheads * dim))
        torch.cuda.synchronize()
        return out[0]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,window,dtype", [((4, 2, 64), 0, "f32"), ((4, 2, 64), 40, "bf16"),
                                                ((2, 1, 256), 40, "f32")],
                         ids=["f32", "window-bf16", "window-d256"])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_a_batch_through_its_life(pcl, torch, heads, window, dtype, captured):
    # prompts, decode steps, idle requests, a step that does not fit, refused
    # speculative tokens, a release and the reuse of its pages; with a graph,
    # every step is a replay of one capture, with other counts
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx = pcl.Context(0, stream.cuda_stream)
    plain = pcl.Context(0, torch.cuda.current_stream().cuda_stream)
    shape = (5, 40, 8, 90, 600)
    server = Server(pcl, torch, ctx, heads, shape[0], shape[2], shape[3], shape[1], shape[4],
                    window, dtype)
    model = PageModel(*shape)
    reference = Reference(server)
    torch.cuda.synchronize()
    graphs = []
    if captured:
        server.step(commit=False)  # no tokens: builds the rotation table
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            server.step(commit=False)
        graphs.append(graph)
    plans = [([300, 0, 7, 1, 0], None, None), ([1, 0, 1, 1, 0], None, None),
             ([1, 257, 0, 1, 0], None, None), ([1, 1, 1, 1, 200], None, None),
             ([5, 4, 3, 2, 1], [1, 4, 0, 2, 0], None), ([1, 1, 1, 1, 1], None, [1, 0, 0, 0, 1]),
             ([250, 1, 0, 1, 1], None, None), ([1, 1, 1, 1, 1], None, None)]
    g = torch.Generator(device="cuda:0")
    g.manual_seed(3)
    for counts, kept, finished in plans:
        for x in server.raw:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda:0"))
        server.batch.put(counts)
        server.attended.fill_(9.5)
        torch.cuda.synchronize()
        ok = model.step(counts)
        if captured:
            graphs[0].replay()
        else:
            server.step(commit=False)
        torch.cuda.synchronize()
        assert ctx.sync() == (0 if ok else BAD_PAGES), counts
        model.check(server.batch.state())
        got = server.attended.clone()
        reference.take(model)
        for b, row in enumerate(model.newest):
            if row >= 0:
                want = reference.attended(b)
                assert np.array_equal(bits(got[row] + 0.0), bits(want + 0.0)), (counts, b)
        idle = torch.ones(shape[4], dtype=torch.bool, device="cuda:0")
        idle[[r for r in model.newest if r >= 0]] = False
        assert bool((got[idle] == 9.5).all())
        # the output block over the same rows
        result = server.result.clone()
        again = [torch.empty_like(result) for _ in range(2)]
        torch.cuda.synchronize()
        plain.attention_output(got.data_ptr(), server.rows, got.shape[1], server.w.data_ptr(),
                               server.hidden, server.post.data_ptr(), 1e-6,
                               server.residual.data_ptr(), again[0].data_ptr(),
                               again[1].data_ptr())
        assert plain.sync() == 0
        assert np.array_equal(bits(result), bits(again[1]))
        ctx.page_commit(server.batch.desc, None if kept is None else server.batch.put(kept))
        torch.cuda.synchronize()
        assert model.commit(kept)
        reference.keep(model.lengths)
        if finished:
            server.batch.put(finished)
            torch.cuda.synchronize()
            ctx.page_release(server.batch.desc, server.batch.words.data_ptr())
            torch.cuda.synchronize()
            model.release(finished)
            reference.keep(model.lengths)
        assert ctx.sync() == 0
        model.check(server.batch.state())
    for graph in graphs:
        graph.reset()
    server.transform.close()
    ctx.close()
    plain.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype", [((12, 1, 128), "bf16"), ((8, 1, 256), "f32"),
                                         ((9, 3, 112), "bf16")], ids=str)
def test_a_first_call_inside_a_capture(pcl, torch, heads, dtype):
    # nothing of a kernel's setup needs a call before the capture
    stream = torch.cuda.Stream()
    cache = Cache(pcl, torch, heads, [300, 5, 900], 16, dtype, 9)
    qheads, _, dim = heads
    q = torch.randn((3, qheads * dim), device="cuda:0")
    out = torch.full_like(q, 9.5)
    torch.cuda.synchronize()
    ctx = pcl.Context(0, stream.cuda_stream)
    d = ctx.paged_desc(
        pools=cache.pools.desc, q=q.data_ptr(), q_stride=qheads * dim, q_rows=3, qheads=qheads,
        table=cache.table.data_ptr(), table_stride=cache.stride,
        lengths=cache.dlengths.data_ptr(), requests=3, max_length=900, q_scale=scale_of(dim),
        out=out.data_ptr(), o_stride=qheads * dim)
    ctx.reserve(ctx.paged_workspace_bytes(d))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.paged_attention(d)
    for i in range(4):
        q.normal_()
        out.fill_(9.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for b in range(3):
            want = cache.contiguous(ctx, q[b:b + 1], b)
            assert np.array_equal(bits(out[b] + 0.0), bits(want + 0.0))
        assert ctx.sync() == 0
    graph.reset()
    ctx.close()


@pytest.mark.gpu
def test_captures_do_not_allocate(pcl, torch):
    # inside a capture a workspace or rotation table that is too small is
    # refused; what a capture holds survives a later growth
    stream = torch.cuda.Stream()
    ctx = pcl.Context(0, stream.cuda_stream)
    heads = (4, 2, 64)
    small = Cache(pcl, torch, heads, [600, 30], 16, "f32", 31)
    q = torch.randn((2, 256), device="cuda:0")
    out = torch.full_like(q, 9.5)
    want = torch.stack([small.contiguous(ctx, q[b:b + 1], b) for b in range(2)])
    assert ctx.sync() == 0
    torch.cuda.synchronize()
    fresh = pcl.Context(0, stream.cuda_stream)
    tr = pcl.HeadTransform(fresh, 4, 2, 64, np.ones(64), np.ones(64), 1e-6, 10000.0)
    d = fresh.paged_desc(
        pools=small.pools.desc, q=q.data_ptr(), q_stride=256, q_rows=2, qheads=4,
        table=small.table.data_ptr(), table_stride=small.stride, lengths=small.dlengths.data_ptr(),
        requests=2, max_length=608, q_scale=scale_of(64), out=out.data_ptr(), o_stride=256)
    slots = torch.tensor([0], dtype=torch.int32, device="cuda:0")
    rows = torch.randn((1, 4, 64), device="cuda:0")
    spare = Pools(pcl, torch, 2, 4, 2, 64, "f32")
    tr_out = torch.empty_like(rows)

    def append():
        tr.append_paged(spare.desc, slots.data_ptr(), slots.data_ptr(), 100, rows.data_ptr(),
                        rows.data_ptr(), rows.data_ptr(), 1, tr_out.data_ptr())

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out.mul_(1.0)  # the capture holds a node either way
        for call in (lambda: fresh.paged_attention(d), append):
            with pytest.raises(pcl.AttentionError) as e:
                call()
            assert e.value.kind == "ResourceLimit"
    torch.cuda.synchronize()
    graph.reset()
    fresh.reserve(fresh.paged_workspace_bytes(d))
    append()
    torch.cuda.synchronize()
    kept = tr_out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        fresh.paged_attention(d)
        append()
    big = Cache(pcl, torch, heads, [30000, 600], 16, "f32", 32)
    q_big = torch.randn((2, 256), device="cuda:0")
    torch.cuda.synchronize()
    for _ in range(4):
        out.fill_(9.5)
        tr_out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(bits(out + 0.0), bits(want + 0.0))
        assert torch.equal(tr_out, kept)
        # grows the workspace and the rotation table
        big.attend(fresh, q_big)
        tr.append_paged(spare.desc, slots.data_ptr(), slots.data_ptr(), 5000, rows.data_ptr(),
                        rows.data_ptr(), rows.data_ptr(), 1, tr_out.data_ptr())
        assert fresh.sync() == 0
    graph.reset()
    tr.close()
    fresh.close()
    ctx.close()
