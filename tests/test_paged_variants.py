"""Every compiled kernel of pcl_paged_tree_attention: which launch takes which, its
bits and error on that launch, and its registers.

A launch's kernel follows from the head dim, the page type, the rows of a KV head that
a request has at most and the items (tree_variant of csrc/paged_tree.hip, which the
tests ask, so that a change of the rule cannot leave a kernel without its test).
"""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import test_paged as tp
from test_paged import bits, ctx, torch  # noqa: F401
from test_paged_tree import TreeCache, random_trees

CUS = 256  # of an MI355X


class Variant(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int), ("buffers", ctypes.c_int)]


def variant_of(pcl, dim, chunks, kvheads, rows, cus=CUS):
    fn = pcl.load()._ZN3pcl12tree_variantElllll
    fn.restype = Variant
    fn.argtypes = [ctypes.c_int64] * 5
    v = fn(dim, chunks, kvheads, rows, cus)
    return v.rows, v.buffers


# query heads of a KV head and the most new tokens of a request, for each unit of rows
SHAPES = {4: (2, 2), 8: (3, 2), 16: (4, 4), 32: (8, 3), 48: (5, 8)}
DIMS = [64, 48, 128, 80, 256, 208, 512, 272]  # whole and padded
KVHEADS = 4
# held tokens around tiles, pages and chunks: of few items, of few in units of eight rows
# (192 over the KV heads) and of many (288)
FEW = [0, 255, 300]
EIGHTS = [33, 200, 255, 256, 500, 700, 1000, 1500]
MANY = [0, 0, 1, 31] + EIGHTS


def padded(dim):
    return next(d for d in (64, 128, 256, 512) if dim <= d)


def cases():
    """(dim, dtype, rows of the unit, buffers, held tokens)."""
    out = []
    for dim in DIMS:
        for dtype in ("f32", "bf16"):
            for unit in SHAPES:
                if unit == 48 and dim > 256:
                    continue
                if unit <= 8 and dim == padded(dim):
                    out.append((dim, dtype, unit, 2, FEW if unit == 4 else EIGHTS))
                out.append((dim, dtype, unit, 1 if unit <= 8 else 0, MANY))
    return out


def launch_of(unit, held):
    """(query heads, new tokens of each request, max_length, chunks of the launch)."""
    group, most = SHAPES[unit]
    counts = [1 + (5 * b + most - 1) % most for b in range(len(held))]
    counts[len(held) // 2] = 0
    counts[1] = most
    length = max(a + n for a, n in zip(held, counts))
    return group * KVHEADS, counts, length, len(held) * -(-length // 256)


def kernel_of(dim, dtype, unit, buffers):
    """A kernel's name without the ring of the many-row ones."""
    kind = "f" if dtype == "f32" else "DF16b"
    whole = int(dim == padded(dim))
    if buffers:
        return "paged_tree %d %s %d %d %d" % (padded(dim), kind, whole, unit // 4, buffers)
    return "tree_rows %d %s %d %d" % (padded(dim), kind, whole, unit // 16)


def test_a_case_for_every_compiled_kernel(pcl):
    pcl.load()
    symbols = subprocess.run(["nm", "-D", "--defined-only", pcl.LIB_PATH], check=True,
                             capture_output=True, text=True).stdout
    compiled = set()
    for name, dk, kind, whole, n, nb in re.findall(
            r"_ZN3pcl\d+(paged_tree|tree_rows)_kernelILi(\d+)E(f|DF16b)Lb([01])ELi(\d)ELi(\d)E",
            symbols):
        compiled.add(" ".join((name, dk, kind, whole, n) + ((nb,) if name == "paged_tree" else ())))
    assert len(compiled) == 48 + 44
    reached = set()
    for dim, dtype, unit, buffers, held in cases():
        group, most = SHAPES[unit]
        chunks = launch_of(unit, held)[3]
        assert variant_of(pcl, dim, chunks, KVHEADS, group * most) == (unit, buffers)
        reached.add(kernel_of(dim, dtype, unit, buffers))
    assert reached == compiled


def test_variants_of_launches(pcl):
    # rows of one unit and of several
    for rows, unit in ((1, 4), (4, 4), (5, 8), (8, 8), (9, 16), (16, 16), (17, 32), (32, 32),
                       (33, 48), (48, 48), (49, 32), (64, 32), (65, 48), (97, 48), (1 << 20, 48)):
        assert variant_of(pcl, 256, 1 << 20, 8, rows) == (unit, 0 if unit > 8 else 1)
        assert variant_of(pcl, 48, 1, 1, rows) == (unit, 0 if unit > 8 else 1)
    for rows, unit in ((9, 16), (16, 16), (17, 32), (33, 32), (49, 32), (1 << 20, 32)):
        assert variant_of(pcl, 512, 1 << 20, 8, rows) == (unit, 0)
    assert variant_of(pcl, 64, 64, 4, 4) == (4, 2)
    assert variant_of(pcl, 64, 65, 4, 4) == (4, 1)
    assert variant_of(pcl, 64, 8, 4, 32) == (4, 2)
    assert variant_of(pcl, 64, 16, 4, 32) == (8, 2)
    assert variant_of(pcl, 64, 17, 4, 32) == (32, 0)
    # few items of padded head dims above 64 have one buffer
    for dim in (80, 112, 144, 208, 272, 496):
        assert variant_of(pcl, dim, 8, 4, 32) == (4, 1)
        assert variant_of(pcl, dim, 16, 4, 32) == (8, 1)
        assert variant_of(pcl, dim, 17, 4, 32) == (32, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(10, 2, 80), (16, 8, 144), (6, 3, 208), (16, 2, 400),
                                   (4, 1, 112), (16, 4, 48)],
                         ids=lambda h: "x".join(map(str, h)))
def test_few_items_of_padded_head_dims(pcl, torch, ctx, dtype, heads):
    qheads, kvheads, dim = heads
    rng = np.random.default_rng(dim)
    for held, counts in (([100], [6]), ([1000], [8]), ([500], [40]), ([64, 2, 700], [9, 4, 12])):
        masks, positions = random_trees(rng, held, counts)
        for tree in (None, masks):
            cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, sum(held), tree,
                              positions if tree else None)
            q = cache.queries()
            length = max(cache.lengths)
            rows = max(counts) * qheads // kvheads
            variant = variant_of(pcl, dim, len(held) * -(-length // 256), kvheads, rows)
            assert variant[1] == (1 if dim > 64 or rows <= 8 else 0)
            for window, softcap in ((0, 0.0), (70, 0.0), (0, 1.5)):
                out = cache.tree_attend(ctx, q, window=window, softcap=softcap,
                                        max_length=length)
                assert ctx.sync() == 0
                cache.check(ctx, q, out, window=window, softcap=softcap)
    assert ctx.sync() == 0


def resources(source):
    """{kernel: (scratch bytes a lane, vector registers spilled)} of a source."""
    import importlib.util
    import tempfile
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "power-cpu-llm_amd")
    spec = importlib.util.spec_from_file_location("hip_build", os.path.join(root, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    with tempfile.TemporaryDirectory() as tmp:
        res = subprocess.run(
            [build.HIPCC] + [f for f in build.FLAGS if f != "-shared"] +
            ["--cuda-device-only", "-c", "-Rpass-analysis=kernel-resource-usage",
             os.path.join(root, "csrc", source), "-o", os.path.join(tmp, "k.o")],
            capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    found = {}
    for line in res.stderr.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        if m:
            words = found.setdefault(m.group(1), {})
        m = re.search(r"(ScratchSize \[bytes/lane\]|VGPRs Spill): (\d+)", line)
        if m:
            words[m.group(1)[0]] = int(m.group(2))
    return {name: (w["S"], w["V"]) for name, w in found.items()}


@pytest.fixture(scope="module")
def compiled():
    """The same of every kernel of the tree attention, by source."""
    from concurrent.futures import ThreadPoolExecutor
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc absent")
    sources = ["paged_%s_d%d.hip" % (kind, dk) for kind in ("rows", "tree")
               for dk in (512, 64, 128, 256)]
    with ThreadPoolExecutor(8) as pool:
        return dict(zip(sources, pool.map(resources, sources)))


def kernels_of(compiled, kind, name):
    return {n: w for s, r in compiled.items() if kind in s for n, w in r.items() if name in n}


def test_no_kernel_of_few_rows_keeps_its_words_in_memory(compiled):
    kernels = kernels_of(compiled, "paged_tree", "paged_tree_kernel")
    assert len(kernels) == 48
    assert {n: w for n, w in kernels.items() if w != (0, 0)} == {}


# registers that spill where both ways around it were slower: 48 rows at padded head dim
# 128 with bf16 pages (the compiler holds 256; a bound of 512 puts sums into AGPRs)
SPILLS = {"_ZN3pcl16tree_rows_kernelILi128EDF16bLb0ELi3ELi3EEEvNS_10TreeParamsE": (32, 8)}


def test_no_kernel_of_many_rows_keeps_its_words_in_memory(compiled):
    kernels = kernels_of(compiled, "paged_rows", "tree_rows_kernel")
    assert len(kernels) == 44 and set(SPILLS) <= set(kernels)
    for name, words in kernels.items():
        most = SPILLS.get(name, (0, 0))
        assert words[0] <= most[0] and words[1] <= most[1], (name, words)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype,unit,buffers,held", cases(),
                         ids=lambda x: None if isinstance(x, list) else str(x))
def test_each_kernel_has_the_contiguous_bits(pcl, torch, ctx, dim, dtype, unit, buffers, held):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    qheads, counts, length, chunks = launch_of(unit, held)
    group, most = SHAPES[unit]
    assert variant_of(pcl, dim, chunks, KVHEADS, group * most, cus) == (unit, buffers)
    masks, positions = random_trees(np.random.default_rng(dim + unit), held, counts)
    for tree in (None, masks):
        cache = TreeCache(pcl, torch, (qheads, KVHEADS, dim), held, counts, 16, dtype, dim, tree,
                          positions if tree else None)
        q = cache.queries()
        for window, softcap in ((0, 0.0), (100, 0.0), (0, 1.5)):
            out = cache.tree_attend(ctx, q, window=window, softcap=softcap, max_length=length,
                                    max_new=most)
            assert ctx.sync() == 0
            cache.check(ctx, q, out, window=window, softcap=softcap, exact=tree is not None)
            assert bool((out[cache.rows - 3:] == 9.5).all())
    assert ctx.sync() == 0


# Whole spans of chunks are items from as many chunks on (over the units and KV heads) as
# the longest span has, for each workgroup: at most four on a CU. Requests of one span of
# three chunks, enough for four workgroups on each CU; and of a whole span of sixteen and a
# part of the next, 8640 chunks for two workgroups a CU (8192).
SPANS = [((32, 8, 64), "f32", 16, [513 + i for i in range(140)]),
         ((32, 8, 128), "f32", 16, [600 - 7 * i % 80 for i in range(140)]),
         ((16, 8, 256), "bf16", 16, [600 + i for i in range(144)]),
         ((16, 8, 256), "f32", 32, [590 + i % 40 for i in range(144)]),
         ((32, 8, 128), "bf16", 32, [513 + i for i in range(140)]),
         ((32, 8, 64), "bf16", 16, [4360 + 3 * i for i in range(60)])]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype,unit,held", SPANS, ids=lambda x: None
                         if isinstance(x, list) else str(x))
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_spans_of_small_units_as_items(pcl, torch, ctx, heads, dtype, unit, held, tree):
    qheads, kvheads, dim = heads
    group = qheads // kvheads
    most = unit // group
    counts = [most - i % 3 for i in range(len(held))]
    masks = positions = None
    if tree:
        masks, positions = random_trees(np.random.default_rng(dim), held, counts)
    cache = TreeCache(pcl, torch, heads, held, counts, 64, dtype, 29, masks, positions)
    length = max(cache.lengths)
    chunks = len(held) * -(-length // 256)
    assert chunks * kvheads >= 3 * 4 * CUS
    assert variant_of(pcl, dim, chunks, kvheads, group * most) == (unit, 0)
    q = cache.queries()
    out = cache.tree_attend(ctx, q, max_length=length)
    assert ctx.sync() == 0
    again = cache.tree_attend(ctx, q, max_length=length)
    assert np.array_equal(bits(out), bits(again))
    cache.check(ctx, q, out, requests=[0, 1, len(held) // 2, len(held) - 2, len(held) - 1],
                exact=False)
    assert bool((out[cache.rows - 3:] == 9.5).all())
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(4, 2, 64), (32, 2, 128), (48, 3, 80)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_scores_of_minus_infinity(pcl, torch, ctx, dtype, heads, tree):
    # a token whose every score is -infinity keeps its row; for one that attends other
    # keys too that key counts for nothing; both set bit 0
    qheads, kvheads, dim = heads
    held, counts = [0, 0, 300], [1, 5, 4]
    masks = positions = None
    if tree:
        masks = [np.tril(np.ones((n, n), bool)) for n in counts]
        positions = [[a + i for i in range(n)] for a, n in zip(held, counts)]
    cache = TreeCache(pcl, torch, heads, held, counts, 16, dtype, 3, masks, positions)
    q = cache.queries()
    q.view(cache.rows, qheads, dim)[:, :, 3] = 1.0
    outs = []
    for bad in (-1e30, float("-inf")):  # (scores far below the others': weights of 0 too)
        for b, at in ((0, 0), (1, 0), (2, 17)):
            slot = int(cache.table[b, at // 16]) * 16 + at % 16
            cache.pools.k.view(-1, kvheads, dim)[slot, :, 3] = bad
        outs.append(cache.tree_attend(ctx, q))
        assert ctx.sync() == (0 if bad > -float("inf") else 1)
    want, out = outs
    alone = [cache.first[0], cache.first[1]]
    assert bool(torch.isfinite(out).all()) and bool((out[alone] == 9.5).all())
    want[alone] = 9.5
    assert np.array_equal(bits(out + 0.0), bits(want + 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4096, 1, 16), (4096, 4096, 16), (4095, 3, 16)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_heads_at_their_bounds(pcl, torch, ctx, heads, tree):
    held, counts = [300, 0, 5], [2, 3, 1]
    masks = positions = None
    if tree:
        masks, positions = random_trees(np.random.default_rng(7), held, counts)
    cache = TreeCache(pcl, torch, heads, held, counts, 16, "bf16", 3, masks, positions)
    q = cache.queries()
    for window in (0, 260):
        out = cache.tree_attend(ctx, q, window=window)
        assert ctx.sync() == 0
        cache.check(ctx, q, out, window=window)
        assert bool((out[cache.rows - 3:] == 9.5).all())
    assert ctx.sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads,new", [((1, 1, 16), 3), ((12, 1, 16), 2)], ids=str)
def test_a_length_bound_far_above_the_lengths(pcl, torch, ctx, heads, new):
    # chunks, partials and items counted from 2^28 and more tokens
    cache = TreeCache(pcl, torch, heads, [700], [new], 16, "f32", 3, rows=new)
    q = cache.queries()
    want = cache.tree_attend(ctx, q)
    for length in (1 << 26, (1 << 28) + 7):
        out = cache.tree_attend(ctx, q, max_length=length, table_stride=1 << 25)
        assert ctx.sync() == 0
        assert np.array_equal(bits(out), bits(want)), length
    cache.check(ctx, q, want)
    assert ctx.sync() == 0
