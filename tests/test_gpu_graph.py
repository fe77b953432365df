"""Device-resident launches captured into a HIP graph (GPU).

A caller that replays a decode step as a graph (torch.cuda.CUDAGraph on the
context's stream) gets, on every replay, the bits the same launch gives
eagerly, with new inputs copied into the captured buffers between replays.
While a stream is capturing, AUTO never picks the spread decode (its
workgroups accept a published word by the launch's epoch, a kernel argument
every replay would repeat): it takes the pipelined kernel, whose bits are the
same, and an explicit spread request is refused. Both the allocating entry
(workspace reserved before the capture) and the allocation-free entry are
captured. Replays are checked against eager launches of the same inputs, with
eager work and synchronisations between the replays.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a GPU"
    return t


def bits(x):
    return np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)


class Step:
    """Device buffers of one decode (Q, K, V, out) and its descriptor."""

    def __init__(self, torch, ctx, qheads, kvh, dim, nkeys, kernel=0):
        dev = torch.device("cuda:0")
        self.q = torch.empty((1, qheads * dim), device=dev)
        self.k = torch.empty((nkeys, kvh, dim), device=dev)
        self.v = torch.empty((nkeys, kvh, dim), device=dev)
        self.out = torch.full((1, qheads * dim), float("nan"), device=dev)
        self.desc = ctx.desc(q=self.q.data_ptr(), q_stride=qheads * dim, nq=1, qheads=qheads,
                             kvheads=kvh, dim=dim, kh_first=0, kh_end=kvh, causal=1,
                             first_query=nkeys - 1, k0=self.k.data_ptr(), v0=self.v.data_ptr(),
                             n0=nkeys, out=self.out.data_ptr(), o_stride=qheads * dim,
                             kernel=kernel, q_scale=float(np.float32(1.0 / np.sqrt(dim))))

    def fill(self, torch, seed):
        g = torch.Generator(device="cuda:0")
        g.manual_seed(seed)
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda:0"))


def eager(torch, pcl, step, kernel=0):
    """The same inputs through an eager launch on torch's current stream."""
    ctx = pcl.Context(0, torch.cuda.current_stream().cuda_stream)
    try:
        out = torch.full_like(step.out, float("nan"))
        d = ctx.desc(**{f: getattr(step.desc, f) for f, _ in step.desc._fields_})
        d.out = out.data_ptr()
        d.kernel = kernel
        ctx.launch(d)
        assert ctx.sync() == 0
        return out.cpu().numpy()
    finally:
        ctx.close()


# a 2K decode (AUTO picks the spread decode eagerly) and a 32K one (the
# pipelined decode and its combine)
GRAPH_CASES = [(16, 8, 256, 2048), (16, 8, 256, 32768)]


@pytest.mark.parametrize("noalloc", [False, True], ids=["launch", "noalloc"])
@pytest.mark.parametrize("case", GRAPH_CASES, ids=lambda c: "x".join(map(str, c)))
def test_graph_replays_give_the_eager_bits(pcl, torch, case, noalloc):
    qheads, kvh, dim, nkeys = case
    stream = torch.cuda.Stream()
    ctx = pcl.Context(0, stream.cuda_stream)
    try:
        step = Step(torch, ctx, qheads, kvh, dim, nkeys)
        step.fill(torch, 0x6A0)
        launch = ctx.launch_noalloc if noalloc else ctx.launch
        torch.cuda.synchronize()
        if not noalloc:
            ctx.reserve(ctx.workspace_bytes(step.desc))
        with torch.cuda.stream(stream):
            launch(step.desc)  # eager on the capture stream first
        stream.synchronize()
        assert ctx.sync() == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            launch(step.desc)
        for rep in range(4):
            step.fill(torch, 0x6A1 + rep)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = step.out.cpu().numpy()
            assert ctx.sync() == 0
            want = eager(torch, pcl, step)
            assert np.array_equal(bits(got), bits(want)), rep
        graph.reset()
    finally:
        ctx.close()


def test_capture_refuses_an_explicit_spread_request(pcl, torch):
    stream = torch.cuda.Stream()
    ctx = pcl.Context(0, stream.cuda_stream)
    try:
        step = Step(torch, ctx, 16, 8, 256, 2048, kernel=pcl.KERNEL_SPREAD_KV)
        step.fill(torch, 0x6B0)
        ctx.reserve(ctx.workspace_bytes(step.desc))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(pcl.AttentionError) as e:
            with torch.cuda.graph(graph, stream=stream):
                step.out.mul_(1.0)  # the capture holds one node either way
                ctx.launch(step.desc)
        assert e.value.kind == "InvalidParameter"
        torch.cuda.synchronize()
        # outside a capture the same request runs, with the pipelined bits
        with torch.cuda.stream(stream):
            ctx.launch(step.desc)
        stream.synchronize()
        assert ctx.sync() == 0
        got = step.out.cpu().numpy()
        want = eager(torch, pcl, step, kernel=pcl.KERNEL_PIPE_KV)
        assert np.array_equal(bits(got), bits(want))
    finally:
        ctx.close()


@pytest.mark.parametrize("n", [1, 4, 20, 40, 200, 700, 1400])
def test_output_block_replays_give_the_eager_bits(pcl, torch, n):
    # every projection form, captured without an eager call on its stream
    cols, rows = 516, 2816
    dev = torch.device("cuda:0")
    stream = torch.cuda.Stream()
    ctx = pcl.Context(0, stream.cuda_stream)
    plain = pcl.Context(0, torch.cuda.current_stream().cuda_stream)
    try:
        x, res = torch.empty((n, cols), device=dev), torch.empty((n, rows), device=dev)
        w = torch.randn((rows, cols), device=dev)
        scale = torch.randn(rows, device=dev)
        proj, out = torch.empty((n, rows), device=dev), torch.empty((n, rows), device=dev)

        def call(c, p, o):
            c.attention_output(x.data_ptr(), n, cols, w.data_ptr(), rows, scale.data_ptr(), 1e-6,
                               res.data_ptr(), p.data_ptr(), o.data_ptr())

        x.normal_()
        res.normal_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(ctx, proj, out)
        for _ in range(4):
            x.normal_()
            res.normal_()
            proj.fill_(float("nan"))
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want_p, want = torch.empty_like(proj), torch.empty_like(out)
            call(plain, want_p, want)
            assert plain.sync() == 0 and ctx.sync() == 0
            assert np.array_equal(bits(proj.cpu().numpy()), bits(want_p.cpu().numpy()))
            assert np.array_equal(bits(out.cpu().numpy()), bits(want.cpu().numpy()))
        graph.reset()
    finally:
        ctx.close()
        plain.close()


def nan_blocks(torch, nbytes, count=24):
    """Fresh device memory full of NaNs, where a freed block of `nbytes` would
    be handed out again."""
    blocks = [torch.full((max(nbytes // 4, 1),), float("nan"), device="cuda:0")
              for _ in range(count)]
    torch.cuda.synchronize()
    return blocks


@pytest.mark.parametrize("grow", ["reserve", "launch", "paged"])
def test_a_captured_launch_keeps_its_workspace(pcl, torch, grow):
    # the graph holds the workspace's address: a later call that needs a larger
    # one leaves the old one to the graph
    stream = torch.cuda.Stream()
    ctx = pcl.Context(0, stream.cuda_stream)
    try:
        step = Step(torch, ctx, 16, 8, 256, 8192, kernel=pcl.KERNEL_PIPE_KV)
        step.fill(torch, 0x6C0)
        held = ctx.workspace_bytes(step.desc)
        ctx.reserve(held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ctx.launch(step.desc)
        if grow == "reserve":
            ctx.reserve(4 * held)
        elif grow == "launch":
            big = Step(torch, ctx, 16, 8, 256, 40000, kernel=pcl.KERNEL_PIPE_KV)
            big.fill(torch, 0x6C1)
            torch.cuda.synchronize()
            ctx.launch(big.desc)
        else:
            k = torch.zeros((64, 256, 8, 256), device="cuda:0")
            pools = pcl.page_pools(k=k.data_ptr(), v=k.data_ptr(), type=pcl.CACHE_F32, pages=64,
                                   page_tokens=256, kvheads=8, dim=256)
            table = torch.arange(64, device="cuda:0", dtype=torch.int32).repeat(4, 1)
            lengths = torch.full((4,), 64 * 256, device="cuda:0", dtype=torch.int32)
            q = torch.zeros((4, 16 * 256), device="cuda:0")
            torch.cuda.synchronize()
            ctx.paged_attention(ctx.paged_desc(
                pools=pools, q=q.data_ptr(), q_stride=16 * 256, q_rows=4, qheads=16,
                table=table.data_ptr(), table_stride=64, lengths=lengths.data_ptr(), requests=4,
                max_length=64 * 256, out=q.data_ptr(), o_stride=16 * 256))
        assert ctx.sync() == 0
        blocks = nan_blocks(torch, held)
        for rep in range(4):
            step.fill(torch, 0x6C2 + rep)
            step.out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = step.out.cpu().numpy()
            assert ctx.sync() == 0
            want = eager(torch, pcl, step, kernel=pcl.KERNEL_PIPE_KV)
            assert np.array_equal(bits(got), bits(want)), rep
            # nobody else's memory was written
            assert all(bool(torch.isnan(b).all()) for b in blocks), rep
        graph.reset()
    finally:
        ctx.close()


@pytest.mark.parametrize("call", ["prepare", "query", "append", "attend_token"])
def test_a_captured_transform_keeps_its_rotation_table(pcl, torch, call):
    # the same of the table of a transform, which grows with the positions; a
    # table that is too short is refused inside a capture, which goes on
    qheads, kvh, dim, at = 16, 8, 256, 40
    stream = torch.cuda.Stream()
    ctx = pcl.Context(0, stream.cuda_stream)
    plain = pcl.Context(0, torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(7)
    scales = [1.0 + 0.1 * rng.standard_normal(dim) for _ in range(2)]
    # prepared queries, keys and values, and the attended output
    shapes = [(1, h, dim) for h in (qheads, kvh, kvh, qheads)]
    made = []

    def side(c):
        """A transform, a cache of `at` tokens and the outputs on context c."""
        t = pcl.HeadTransform(c, qheads, kvh, dim, *scales, 1e-6, 10000.0)
        cache = pcl.LayerCache(c, kvh, dim, 1 << 20, None, 1 << 30)
        cache.reserve_rows(1024)
        rows = torch.full((at, kvh, dim), 0.5, device="cuda:0")
        torch.cuda.synchronize()
        cache.append(rows.data_ptr(), rows.data_ptr(), at)
        cache.commit()
        assert c.sync() == 0
        out = [torch.full(s, float("nan"), device="cuda:0") for s in shapes]
        made.extend((cache, t))
        return t, cache, out

    def run(t, cache, out):
        ptr = [x.data_ptr() for x in raw + out]
        if call == "prepare":
            t.prepare(*ptr[:3], 1, at, *ptr[3:6])
        elif call == "query":
            t.query(ptr[0], 1, at, ptr[3])
        elif call == "append":
            cache.append_transformed(t, *ptr[:3], 1, ptr[3])
        else:
            cache.attend_token(t, *ptr[:3], ptr[3], ptr[6], q_scale=0.0625)

    try:
        raw = [torch.randn(s, device="cuda:0") for s in shapes[:3]]
        t, cache, out = side(ctx)
        ctx.reserve(1 << 24)
        t.query(raw[0].data_ptr(), 1, 0, out[0].data_ptr())  # builds the first rows
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out[3].mul_(1.0)
            with pytest.raises(pcl.AttentionError) as e:
                t.query(raw[0].data_ptr(), 1, 4000, out[0].data_ptr())
            assert e.value.kind == "ResourceLimit"
            run(t, cache, out)
        # a far position: a longer table
        t.query(raw[0].data_ptr(), 1, 5000, out[0].data_ptr())
        assert ctx.sync() == 0
        blocks = nan_blocks(torch, 256 * dim * 4)
        for rep in range(4):
            for x in raw:
                x.normal_()
            for x in out:
                x.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert ctx.sync() == 0
            t2, cache2, want = side(plain)
            run(t2, cache2, want)
            assert plain.sync() == 0
            for got, x in zip(out, want):
                assert np.array_equal(bits(got.cpu().numpy()), bits(x.cpu().numpy())), rep
            if call in ("append", "attend_token"):
                # the appended row (the replay writes it where the capture did)
                for got, x in zip(cache.read(at, 1), cache2.read(at, 1)):
                    assert np.array_equal(bits(got), bits(x)), rep
            assert all(bool(torch.isnan(b).all()) for b in blocks), rep
        graph.reset()
    finally:
        for x in made:
            x.close()
        ctx.close()
        plain.close()
