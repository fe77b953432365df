"""Timing cases of drafted tokens and shared pages over a paged KV cache.

Each case is a plain dict; `kind` names the calls that a program makes in a round
of drafted tokens, or where requests share pages:

  tree    the bookkeeping of a round of drafted trees: Context.page_tree (each
          new token's position and the new tokens before it on its branch) and,
          with the verified branches, Context.page_accept (which rows move where)
  attend  Context.paged_tree_attention: every new token of every request over the
          request's pages, trees by their masks, chains and parts of prompts
          without
  copy    Context.paged_copy: rows of pages moved or copied in all layers at once,
          a verified branch's to its place or a fork's last page to its own
  fork    Context.page_fork, page_commit and page_release_shared: requests that
          begin as copies of others, and their pages given back

`run` makes these calls where `own` is set and computes the same from elementary
torch operations where it is not. Heads, pages and lengths are those of the paged
cases beside this file (16 query and 8 KV heads of 256 dims, sliding layers with a
1024-key window; 16 and 2 of 512), and other heads that the entries accept.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SLIDING = (16, 8, 256)
GLOBAL = (16, 2, 512)
SPARE_PAGES = 5
_contexts = {}


# ---- cases ------------------------------------------------------------------

def _tree(requests, longest, drafts, page, idle=0):
    return {"kind": "tree", "requests": requests, "longest": longest, "drafts": drafts,
            "page": page, "idle": idle}


def _attend(heads, requests, shortest, longest, fewest, drafts, page, dtype, tree=True, window=0,
            idle=0, softcap=0.0):
    qheads, kvheads, dim = heads
    return {"kind": "attend", "qheads": qheads, "kvheads": kvheads, "dim": dim,
            "requests": requests, "shortest": shortest, "longest": longest, "fewest": fewest,
            "drafts": drafts, "page": page, "dtype": dtype, "tree": tree, "window": window,
            "idle": idle, "softcap": softcap}


def _copy(heads, layers, lists, entries, longest, page, dtype):
    _, kvheads, dim = heads
    return {"kind": "copy", "kvheads": kvheads, "dim": dim, "layers": layers, "lists": lists,
            "entries": entries, "longest": longest, "page": page, "dtype": dtype}


def _fork(requests, sources, longest, page):
    return {"kind": "fork", "requests": requests, "sources": sources, "longest": longest,
            "page": page}


def listed():
    return [
        # a small batch's round of drafted trees: launch latency counts
        {"name": "tree_16x12", **_tree(16, 8192, 12, 16)},
        # a full server's round, wide trees, some slots of the batch idle
        {"name": "tree_256x64", **_tree(256, 8192, 64, 16, idle=19)},
        # one young conversation and a short tree: every part of the latency shows
        {"name": "attend_1x6_over_200", **_attend(SLIDING, 1, 200, 200, 6, 6, 16, "f32")},
        # trees of conversations of very different lengths, two slots idle
        {"name": "attend_64x8_over_8k_bf16",
         **_attend(SLIDING, 64, 64, 8192, 5, 8, 16, "bf16", idle=2)},
        # a sliding layer: the window starts inside pages and key chunks
        {"name": "attend_32x24_window",
         **_attend(SLIDING, 32, 2000, 16384, 9, 24, 16, "f32", window=1024)},
        # a global layer, eight query heads to a KV head
        {"name": "attend_16x12_over_32k_d512",
         **_attend(GLOBAL, 16, 2048, 32768, 12, 12, 64, "f32")},
        # short chats with a chain of drafted tokens each
        {"name": "attend_256x4_over_2k_d128_bf16",
         **_attend((32, 8, 128), 256, 16, 2048, 1, 4, 16, "bf16", tree=False, idle=7)},
        # later parts of four prompts behind what their pages hold: the most work
        {"name": "attend_4x512_over_8k",
         **_attend(SLIDING, 4, 1000, 8192, 300, 512, 32, "bf16", tree=False)},
        # the verified branches of 64 requests to their places, six layers
        {"name": "copy_branches_64x5", **_copy(SLIDING, 6, 64, 5, 64, 16, "bf16")},
        # the partly filled last pages of 192 forks, a global layer and two sliding
        # layers' worth of rows
        {"name": "copy_pages_192_d512", **_copy(GLOBAL, 4, 192, 1, 64, 64, "f32")},
        # four answers to each of eight prompts
        {"name": "fork_8x4", **_fork(40, 8, 4000, 16)},
        # many beams over long prompts with small pages: the most pages shared
        {"name": "fork_16x30", **_fork(496, 16, 8192, 8)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = (SLIDING, SLIDING, GLOBAL, (32, 8, 128), (16, 4, 64), (10, 2, 80), (32, 1, 128))


def draw(rng):
    """One more case: sizes over the logarithm of each range."""
    while True:
        kind = rng.choice(("tree", "attend", "attend", "attend", "copy", "fork"))
        page = rng.choice((8, 16, 16, 32, 48, 64, 128))
        dtype = rng.choice(("f32", "bf16"))
        if kind == "tree":
            requests = _log(rng, 1, 512)
            case = _tree(requests, _log(rng, 16, 16384), _log(rng, 2, 200), page,
                         rng.choice((0, requests // 9)))
            if requests * case["drafts"] ** 2 > 1 << 20 or requests * case["longest"] > 1 << 22:
                continue
        elif kind == "attend":
            heads = rng.choice(HEADS)
            tree = rng.choice((True, True, False))
            drafts = _log(rng, 1, 128) if tree else _log(rng, 1, 700)
            longest = _log(rng, 16, 32768)
            requests = _log(rng, 1, 256)
            case = _attend(heads, requests, max(1, longest // rng.choice((1, 4, 64))), longest,
                           max(1, drafts // rng.choice((1, 3))), drafts, page, dtype, tree,
                           window=rng.choice((0, 0, 0, 1024)),
                           idle=rng.choice((0, requests // 9)),
                           softcap=rng.choice((0.0, 0.0, 0.0, 50.0)))
            span = longest + drafts
            if requests * span * heads[1] * heads[2] > 1 << 29 or \
                    requests * span * heads[0] * drafts > 1 << 28 or \
                    work(case)["bytes"] > 1.7e9 or work(case)["flops"] > 1e11:
                continue
        elif kind == "copy":
            entries = rng.choice((1, 1, _log(rng, 2, 12)))
            case = _copy(rng.choice(HEADS), rng.randint(1, 12), _log(rng, 1, 256), entries,
                         _log(rng, 16, 64), page, dtype)
            if work(case)["bytes"] > 1.0e9:
                continue
        else:
            sources = _log(rng, 1, 32)
            case = _fork(sources * rng.randint(2, 33), sources, _log(rng, 16, 8192), page)
            if case["requests"] * case["longest"] // page > 1 << 19:
                continue
        return case


# ---- a case's lengths and trees (the same for every seed) --------------------

def _spread(n, low, high):
    """n lengths spread over the logarithm of [low, high], high among them."""
    i = np.arange(n)
    x = np.round(low * (high / low) ** ((0.6180339887498949 * i + 0.37) % 1.0)).astype(np.int64)
    if n:
        x[n // 2] = high
    return x


def _pages(lengths, page):
    return -(-np.asarray(lengths) // page)


def _parents(counts):
    """Each new token's parent among its request's: one of the four before it,
    or -1 where it follows the held tokens."""
    out = []
    for b, n in enumerate(counts):
        i = np.arange(n)
        out.append(np.maximum(i - 1 - (7 * i + 3 * b) % 4, -1))
    return np.concatenate(out) if out else np.zeros(0, np.int64)


def _idle(requests, idle):
    """Idle slots lie among the others."""
    off = np.zeros(requests, bool)
    if idle:
        off[np.arange(idle) * (requests // idle)] = True
    return off


def _step_of(case):
    """(held tokens, new tokens) of every request."""
    b = case["requests"]
    off = _idle(b, case["idle"])
    if case["kind"] == "tree":
        held = _spread(b, 1, case["longest"])
        counts = _spread(b, max(1, case["drafts"] // 3), case["drafts"])
    else:
        held = _spread(b, case["shortest"], case["longest"])
        counts = _spread(b, case["fewest"], case["drafts"])
    counts[off] = 0
    return held, counts


def _words(case):
    return -(-case["drafts"] // 64)


def _branches(counts, depth):
    """Of each request the branch to one of its last tokens, from the held tokens
    on: (indexes [requests][depth], how many)."""
    paths = np.full((len(counts), depth), -1, np.int64)
    lengths = np.zeros(len(counts), np.int64)
    parents, start = _parents(counts), 0
    for b, n in enumerate(counts):
        mine = parents[start:start + n]
        start += n
        branch, at = [], n - 1 - b % 3
        while at >= 0:
            branch.append(at)
            at = mine[at]
        branch = branch[::-1][:depth]
        paths[b, :len(branch)] = branch
        lengths[b] = len(branch)
    return paths, lengths


def _branch_depth(case):
    return max(1, case["drafts"] // 2)


def _fork_of(case):
    """(tokens held, source of each request or -1): the sources come first, the
    others are free slots that begin as copies, in turn."""
    b, n = case["requests"], case["sources"]
    held = np.zeros(b, np.int64)
    held[:n] = _spread(n, max(1, case["longest"] // 8), case["longest"])
    source = np.full(b, -1, np.int64)
    source[n:] = np.arange(b - n) % n
    return held, source


def _copy_of(case):
    """Rows that each entry copies, [lists][entries]."""
    lists, entries, page = case["lists"], case["entries"], case["page"]
    if entries == 1:
        return (1 + (37 * np.arange(lists) + page // 2) % max(1, page - 1))[:, None]
    some = 1 + np.arange(lists) % entries  # a branch of one token up to all
    return (np.arange(entries)[None, :] < some[:, None]).astype(np.int64)


# ---- inputs -----------------------------------------------------------------

def _package():
    name = "power_cpu_llm_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(ROOT, "power-cpu-llm_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _context():
    """The context that a program keeps for the stream it works on."""
    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _contexts:
        _contexts[stream] = _package().Context(torch.cuda.current_device(), stream)
    return _contexts[stream]


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _table(lengths, stride, page, rng, spare):
    """Block tables over a random order of the pages; -1 where none is held.
    Returns (table, the pages that are left)."""
    held = _pages(lengths, page)
    order = rng.permutation(int(held.sum()) + spare).astype(np.int32)
    table = np.full((len(lengths), stride), -1, np.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    return table, order[at:]


def _types(dtype):
    return torch.float32 if dtype == "f32" else torch.bfloat16


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"case": case}
    {"tree": _prepare_tree, "attend": _prepare_attend, "copy": _prepare_copy,
     "fork": _prepare_fork}[case["kind"]](state, rng, randn)
    return state


BATCH = ("lengths", "table", "free_pages", "counters", "step_lengths", "newest", "slots",
         "positions", "row_request")


def _batch(state):
    case = state["case"]
    return _package().page_batch(
        requests=case["requests"], table_stride=state["stride"], page_tokens=case["page"],
        pages=state["pages"], step_rows=state["rows"],
        **{n: state[n].data_ptr() for n in BATCH})


def _prepare_tree(state, rng, randn):
    """A standing step of drafted tokens, their tree and what was verified."""
    case = state["case"]
    page, b = case["page"], case["requests"]
    held, counts = _step_of(case)
    after = held + counts
    stride = int(_pages(after, page).max()) + 2
    table, free = _table(after, stride, page, rng, SPARE_PAGES)
    n = int(counts.sum())
    rows = n + 7  # a captured step has room for more rows than most steps use
    request = np.repeat(np.arange(b), counts)
    index = np.arange(n) - np.repeat(counts.cumsum() - counts, counts)
    position = held[request] + index
    slots = np.full(rows, -1, np.int64)
    slots[:n] = table[request, position // page].astype(np.int64) * page + position % page
    row_request, sequential = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    row_request[:n], sequential[:n] = request, position
    parents = np.full(rows, -1, np.int64)
    parents[:n] = _parents(counts)
    depth = _branch_depth(case)
    paths, verified = _branches(counts, depth)
    verified = np.minimum(verified, rng.integers(0, depth + 1, b))
    taken = int((_pages(after, page) - _pages(held, page)).sum())
    pages = int(_pages(after, page).sum()) + SPARE_PAGES
    free_pages = np.full(pages, -1, np.int32)
    free_pages[:len(free)] = free
    state.update(pages=pages, rows=rows, stride=stride, depth=depth, words=_words(case),
                 lengths=_ints(held), table=_ints(table), free_pages=_ints(free_pages),
                 counters=_ints([len(free) + taken, n, taken, 1]), step_lengths=_ints(after),
                 newest=_ints(np.where(counts > 0, counts.cumsum() - 1, -1)), slots=_ints(slots),
                 positions=_ints(sequential), row_request=_ints(row_request),
                 parents=_ints(parents), paths=_ints(paths), verified=_ints(verified),
                 moved_from=_ints(np.zeros((b, depth))), moved_to=_ints(np.zeros((b, depth))),
                 tree_positions=_ints(np.zeros(rows)),
                 masks=torch.zeros(rows, _words(case), dtype=torch.int64, device="cuda"))
    if own:
        state["batch"] = _batch(state)
        state["tree"] = _package().page_tree(
            parents=state["parents"].data_ptr(), words=state["words"],
            positions=state["tree_positions"].data_ptr(), masks=state["masks"].data_ptr())


def _ancestors(counts, parents, words):
    """(depth, masks [rows][words]) of the rows' trees."""
    depth = np.zeros(len(parents), np.int64)
    masks = np.zeros((len(parents), words), np.uint64)
    start = 0
    for n in counts:
        for i in range(start, start + n):
            j = parents[i]
            if j >= 0:
                depth[i] = depth[start + j] + 1
                masks[i] = masks[start + j]
            masks[i, (i - start) // 64] |= np.uint64(1) << np.uint64((i - start) % 64)
        start += n
    return depth, masks.view(np.int64)


def _prepare_attend(state, rng, randn):
    case = state["case"]
    page, qheads, kvheads, dim = case["page"], case["qheads"], case["kvheads"], case["dim"]
    held, counts = _step_of(case)
    after = held + counts
    stride = int(_pages(case["longest"] + case["drafts"], page)) + 2
    table, _ = _table(after, stride, page, rng, SPARE_PAGES)
    pages = int(_pages(after, page).sum()) + SPARE_PAGES
    n = int(counts.sum())
    rows = n + 3
    dtype = _types(case["dtype"])
    state.update(pages=pages, stride=stride, rows=rows, words=_words(case),
                 scale=float(np.float32(1.0 / math.sqrt(dim))),
                 lengths=_ints(held), step_lengths=_ints(after),
                 newest=_ints(np.where(counts > 0, counts.cumsum() - 1, -1)), table=_ints(table),
                 k_pages=randn(pages, page, kvheads, dim, dtype=dtype),
                 v_pages=randn(pages, page, kvheads, dim, dtype=dtype),
                 q=randn(rows, qheads * dim), out=torch.zeros(rows + 1, qheads * dim,
                                                              device="cuda"))
    if case["tree"]:
        depth, masks = _ancestors(counts, _parents(counts), state["words"])
        positions = np.full(rows, -1, np.int64)
        positions[:n] = np.repeat(held, counts) + depth
        state["positions"] = _ints(positions)
        state["masks"] = torch.zeros(rows, state["words"], dtype=torch.int64, device="cuda")
        state["masks"][:n] = torch.from_numpy(masks).cuda()
    if own:
        context = _context()
        tree = {}
        if case["tree"]:
            tree = {"masks": state["masks"].data_ptr(), "mask_words": state["words"],
                    "positions": state["positions"].data_ptr()}
        state["desc"] = context.paged_tree_desc(
            pools=_pools(state, "k_pages", "v_pages"), q=state["q"].data_ptr(),
            q_stride=qheads * dim, q_rows=rows, qheads=qheads, table=state["table"].data_ptr(),
            table_stride=stride, lengths=state["lengths"].data_ptr(),
            step_lengths=state["step_lengths"].data_ptr(), newest=state["newest"].data_ptr(),
            requests=case["requests"], max_length=case["longest"] + case["drafts"],
            max_new=case["drafts"], window=case["window"], q_scale=state["scale"],
            softcap=case["softcap"], out=state["out"].data_ptr(), o_stride=qheads * dim, **tree)
        context.reserve(context.paged_tree_workspace_bytes(state["desc"]))


def _pools(state, k, v):
    case = state["case"]
    pcl = _package()
    return pcl.page_pools(
        k=state[k].data_ptr(), v=state[v].data_ptr(),
        type=pcl.CACHE_F32 if case["dtype"] == "f32" else pcl.CACHE_BF16, pages=state["pages"],
        page_tokens=case["page"], kvheads=case["kvheads"], dim=case["dim"])


def _prepare_copy(state, rng, randn):
    """Lists of rows to move: a branch's in the pages of its request, to the rows
    that follow the held ones; or a fork's, one page's first rows to another."""
    case = state["case"]
    page, lists, entries = case["page"], case["lists"], case["entries"]
    rows = _copy_of(case)
    each = 2 if entries == 1 else int(_pages(case["longest"] + 4 * entries, page))
    pages = lists * each + SPARE_PAGES
    order = rng.permutation(pages)[:lists * each].reshape(lists, each)
    if entries == 1:
        source, target = order[:, :1] * page, order[:, 1:] * page
    else:
        # the branch's tokens lie behind as many rows as it may have
        first = (13 * np.arange(lists) % case["longest"])[:, None]
        i = np.arange(entries)[None, :]
        at = first + entries + i * (1 + np.arange(lists)[:, None] % 3)
        source, target = (np.take_along_axis(order, x // page, 1) * page + x % page
                          for x in (at, first + i))
        source = np.where(rows > 0, source, -1)
    dtype = _types(case["dtype"])
    shape = (pages, page, case["kvheads"], case["dim"])
    state.update(pages=pages, source=_ints(source), target=_ints(target), counts=_ints(rows))
    for i in range(case["layers"]):
        state["k%d" % i], state["v%d" % i] = randn(*shape, dtype=dtype), randn(*shape, dtype=dtype)
    if own:
        state["pools"] = [_pools(state, "k%d" % i, "v%d" % i) for i in range(case["layers"])]


def _prepare_fork(state, rng, randn):
    case = state["case"]
    page, b = case["page"], case["requests"]
    held, source = _fork_of(case)
    stride = int(_pages(held, page).max()) + 1
    forks = source >= 0
    need = int((held[source[forks]] % page > 0).sum())
    table, free = _table(held, stride, page, rng, need + SPARE_PAGES)
    free = np.sort(free)[::-1]
    pages = int(_pages(held, page).sum()) + need + SPARE_PAGES
    free_pages = np.full(pages, -1, np.int32)
    free_pages[:len(free)] = free
    rows = b + 9
    state.update(pages=pages, rows=rows, stride=stride, free=len(free), lengths=_ints(held),
                 table=_ints(table), free_pages=_ints(free_pages),
                 counters=_ints([len(free), 0, 0, 0]), source=_ints(source),
                 forks=_ints(forks.astype(np.int64)))
    for name in ("step_lengths", "newest", "copy_from", "copy_to", "copy_rows"):
        state[name] = _ints(np.zeros(b))
    for name in ("slots", "positions", "row_request"):
        state[name] = _ints(np.zeros(rows))
    if own:
        state["batch"] = _batch(state)


# ---- one pass ---------------------------------------------------------------

def run(state):
    return {"tree": _run_tree, "attend": _run_attend, "copy": _run_copy,
            "fork": _run_fork}[state["case"]["kind"]](state)


def _run_tree(state):
    names = ("tree_positions", "masks", "moved_from", "moved_to")
    if own:
        context = _context()
        context.page_tree(state["batch"], state["tree"])
        context.page_accept(state["batch"], state["paths"].data_ptr(),
                            state["verified"].data_ptr(), state["depth"],
                            state["moved_from"].data_ptr(), state["moved_to"].data_ptr())
        return [state[n] for n in names]
    case = state["case"]
    page, words, n = case["page"], state["words"], case["drafts"]
    held, after = state["lengths"].long(), state["step_lengths"].long()
    counts = after - held
    first = state["newest"].long() + 1 - counts
    i = torch.arange(n, device="cuda")
    inside = i < counts[:, None]
    row = torch.where(inside, first[:, None] + i, state["rows"] - 1)
    parent = torch.where(inside, state["parents"][row].long(), -1)
    # which tokens lie on a token's branch: steps to the parent, doubled
    reach = ((parent[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    depth = reach.sum(-1).long() - 1
    bits = torch.zeros(case["requests"], n, 64 * words, dtype=torch.int64, device="cuda")
    bits[:, :, :n] = reach.long()
    masks = (bits.view(case["requests"], n, words, 64) << torch.arange(64, device="cuda")).sum(-1)
    # rows behind the last have no token (a token's row is never the last one)
    state["tree_positions"].fill_(-1)
    state["masks"].zero_()
    state["tree_positions"][row] = torch.where(inside, held[:, None] + depth, -1).int()
    state["masks"][row] = torch.where(inside[:, :, None], masks, 0)
    # a verified token's row moves to the position behind the one before it
    k = torch.arange(state["depth"], device="cuda")
    path = state["paths"].long()
    moves = (k < state["verified"].long()[:, None]) & (path != k)
    for name, index in (("moved_from", path), ("moved_to", k.expand_as(path))):
        position = torch.where(moves, held[:, None] + index, 0)
        slot = state["table"].long().gather(1, position // page) * page + position % page
        state[name].copy_(torch.where(moves, slot, -1))
    return [state[n] for n in names]


def _run_attend(state):
    case = state["case"]
    if own:
        _context().paged_tree_attention(state["desc"])
        return state["out"][:-1]
    page, qheads, kvheads, dim = case["page"], case["qheads"], case["kvheads"], case["dim"]
    b, n, window, words = case["requests"], case["drafts"], case["window"], state["words"]
    group = qheads // kvheads
    held, after = state["lengths"].long(), state["step_lengths"].long()
    counts = after - held
    i = torch.arange(n, device="cuda")
    inside = i < counts[:, None]
    row = torch.where(inside, (state["newest"].long() + 1 - counts)[:, None] + i, state["rows"])
    safe = row.clamp(max=state["rows"] - 1)
    # the keys that any of a request's new tokens attends, and their slots
    span = case["longest"] + n
    if window:
        span = min(span, window + n)
    first = (held + 1 - window).clamp(min=0) if window else torch.zeros_like(held)
    key = first[:, None] + torch.arange(span, device="cuda")
    key = torch.where(key < after[:, None], key, -1)
    slot = state["table"].gather(1, key.clamp(min=0) // page).clamp(min=0).long() * page + \
        key.clamp(min=0) % page
    new = key - held[:, None]  # index among the new tokens
    if case["tree"]:
        own_position = state["positions"][safe].long()
        word = state["masks"][safe].gather(
            2, (new.clamp(0, 64 * words - 1) // 64)[:, None, :].expand(b, n, span))
        bit = (word >> (new.clamp(min=0) % 64)[:, None, :]) & 1
        allowed = torch.where((new < 0)[:, None, :], True, bit == 1)
        at = torch.where(new >= 0, own_position.gather(1, new.clamp(0, n - 1)), key)
    else:
        own_position = held[:, None] + i
        allowed = new[:, None, :] <= i[:, None]
        at = key
    allowed = allowed & (key >= 0)[:, None, :]
    if window:
        allowed = allowed & (own_position[:, :, None] - at[:, None, :] < window)
    q = (state["q"][safe].view(b, n, kvheads, group, dim) * state["scale"]) \
        .permute(0, 2, 1, 3, 4).reshape(b, kvheads, n * group, dim)
    k = state["k_pages"].view(-1, kvheads, dim)[slot].float().permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(q, k)
    del k
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    score = score.view(b, kvheads, n, group, span).masked_fill(~allowed[:, None, :, None, :],
                                                              -math.inf)
    score = score.view(b, kvheads, n * group, span)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    v = state["v_pages"].view(-1, kvheads, dim)[slot].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(weight, v) / weight.sum(-1, keepdim=True)
    # places without a token write the row behind the last
    state["out"][row.view(-1)] = out.view(b, kvheads, n, group, dim).permute(0, 2, 1, 3, 4) \
        .reshape(b * n, qheads * dim)
    return state["out"][:-1]


def _run_copy(state):
    case = state["case"]
    pools = [state[x + str(i)] for i in range(case["layers"]) for x in "kv"]
    if own:
        rows = state["counts"].data_ptr() if case["entries"] == 1 else None
        _context().paged_copy(state["pools"], state["source"].data_ptr(),
                              state["target"].data_ptr(), case["lists"], case["entries"], rows)
        return pools
    i = torch.arange(case["page"] if case["entries"] == 1 else 1, device="cuda")
    real = (i < state["counts"].view(-1, 1)).view(-1)
    source, target = ((state[x].view(-1, 1).long() + i).view(-1) for x in ("source", "target"))
    # places without a row repeat the first row's copy
    source, target = (torch.where(real, x, x[0]) for x in (source, target))
    for x in pools:
        flat = x.view(-1, case["kvheads"], case["dim"])
        flat[target] = flat[source]
    return pools


def _run_fork(state):
    case = state["case"]
    free = state["free"]
    if own:
        context, batch = _context(), state["batch"]
        context.page_fork(batch, state["source"].data_ptr(), state["copy_from"].data_ptr(),
                          state["copy_to"].data_ptr(), state["copy_rows"].data_ptr())
        context.page_commit(batch)
        context.page_release_shared(batch, state["forks"].data_ptr())
    else:
        page, pages = case["page"], state["pages"]
        source = state["source"].long()
        fork = source >= 0
        length = torch.where(fork, state["lengths"][source.clamp(min=0)].long(), 0)
        rest, whole = length % page, length // page
        need = (rest > 0).long()
        order = need.cumsum(0)
        count = state["counters"][0].long()
        fresh = state["free_pages"][(count - order).clamp(min=0)].long()
        # the source's whole pages, and a page of its own for the rest
        column = torch.arange(state["stride"], device="cuda")
        theirs = state["table"][source.clamp(min=0)].long()
        table = torch.where(column < whole[:, None], theirs, state["table"].long())
        last = (need > 0)[:, None] & (column == whole[:, None])
        table = torch.where(fork[:, None], torch.where(last, fresh[:, None], table),
                            state["table"].long())
        state["table"].copy_(table)
        old = theirs.gather(1, whole[:, None].clamp(max=state["stride"] - 1))[:, 0]
        state["copy_from"].copy_(torch.where(need > 0, old * page, -1))
        state["copy_to"].copy_(torch.where(need > 0, fresh * page, -1))
        state["copy_rows"].copy_(rest)
        # held by the forks, and by the others; a commit puts the forks' lengths in
        after = torch.where(fork, length, state["lengths"].long())
        count = count - order[-1]
        held = column < ((after + page - 1) // page)[:, None]
        marks = torch.zeros(2, pages + 1, dtype=torch.int64, device="cuda")
        for mark, who in zip(marks, (fork, ~fork)):
            mark[torch.where(held & who[:, None], table, pages).view(-1)] = 1
        back = ((marks[0] > 0) & (marks[1] == 0))[:pages]
        # they go back highest first
        order = back.flip(0).long().cumsum(0).flip(0)
        grown = torch.cat((state["free_pages"], state["free_pages"][:1]))
        grown[torch.where(back, count + order - 1, pages)] = \
            torch.arange(pages, dtype=torch.int32, device="cuda")
        state["free_pages"].copy_(grown[:pages])
        state["counters"][0] = count + back.long().sum()
        state["lengths"].copy_(torch.where(fork, 0, after))
    return [state[n] for n in ("table", "lengths", "copy_from", "copy_to", "copy_rows")] + \
        [state["counters"][:1], state["free_pages"][:free]]


# ---- what a pass cannot do without, and its result in 64 bits ---------------

def work(case):
    if case["kind"] == "tree":
        _, counts = _step_of(case)
        n, b, depth = int(counts.sum()), case["requests"], _branch_depth(case)
        # lengths and newest rows, parents, paths and counts read, a word of the
        # table for each move; positions, masks and moves written
        return {"bytes": 12 * b + 4 * n + b * (4 * depth + 4) + 4 * b * depth +
                (n + 7) * (4 + 8 * _words(case)) + 8 * b * depth, "flops": n}
    if case["kind"] == "fork":
        held, source = _fork_of(case)
        forks = source >= 0
        pages = _pages(held, case["page"])
        # lengths, sources, the sources' entries and every held one read; the
        # forks' entries, their lengths and copies written
        shared = int(pages[source[forks]].sum())
        return {"bytes": 20 * case["requests"] + 4 * int(pages.sum()) + 8 * shared +
                16 * int(forks.sum()), "flops": shared}
    size = 4 if case["dtype"] == "f32" else 2
    width = case["kvheads"] * case["dim"]
    if case["kind"] == "copy":
        rows = int(_copy_of(case).sum())
        return {"bytes": 4 * size * width * rows * case["layers"] +
                12 * case["lists"] * case["entries"], "flops": 0}
    held, counts = _step_of(case)
    window = case["window"]
    active = counts > 0
    first = np.maximum(held + 1 - window, 0) if window else np.zeros_like(held)
    keys = np.where(active, held + counts - first, 0)
    q = case["qheads"] * case["dim"]
    n = int(counts.sum())
    # (token, key) pairs: the held keys that a token sees and its branch
    if case["tree"]:
        depth, _ = _ancestors(counts, _parents(counts), _words(case))
    else:
        depth = np.arange(n) - np.repeat(counts.cumsum() - counts, counts)
    pairs = np.repeat(held, counts) + depth + 1
    if window:
        pairs = np.minimum(pairs, window)
    return {"bytes": 2 * size * width * int(keys.sum()) +
            4 * int(_pages(keys, case["page"]).sum()) + 8 * q * n + 12 * case["requests"] +
            (n * (8 * _words(case) + 4) if case["tree"] else 0),
            "flops": 4 * q * int(pairs.sum())}


def exact(case, seed):
    if case["kind"] in ("tree", "fork"):
        return None
    state = prepare(case, seed)
    if case["kind"] == "copy":
        return _exact_copy(state)
    return _exact_attend(state)


def _exact_copy(state):
    case = state["case"]
    source, target, rows = (state[x].cpu().numpy().reshape(-1)
                            for x in ("source", "target", "counts"))
    out = []
    for i in range(case["layers"]):
        for x in "kv":
            wide = state[x + str(i)].double().view(-1, case["kvheads"], case["dim"])
            old = wide.clone()
            for a, b, n in zip(source, target, rows):
                wide[b:b + n] = old[a:a + n]
            out.append(wide.view(state[x + str(i)].shape))
    return out


def _exact_attend(state):
    case = state["case"]
    page, qheads, kvheads, dim = case["page"], case["qheads"], case["kvheads"], case["dim"]
    group, window = qheads // kvheads, case["window"]
    held, counts = _step_of(case)
    parents = _parents(counts) if case["tree"] else None
    out = torch.zeros(state["rows"], qheads * dim, dtype=torch.float64, device="cuda")
    row = 0
    for b, (length, n) in enumerate(zip(held.tolist(), counts.tolist())):
        if n == 0:
            continue
        # which keys each new token sees, from the tree itself
        sees = np.zeros((n, length + n), bool)
        sees[:, :length] = True
        position = np.concatenate((np.arange(length), np.zeros(n, np.int64)))
        for i in range(n):
            if parents is None:
                sees[i, length:length + i + 1] = True
                position[length + i] = length + i
                continue
            at, steps = i, 0
            while at >= 0:
                sees[i, length + at] = True
                at, steps = int(parents[row + at]), steps + 1
            position[length + i] = length + steps - 1
        if window:
            sees &= position[length:, None] - position[None, :] < window
        first = int(np.flatnonzero(sees.any(0))[0])
        sees = torch.from_numpy(sees[:, first:]).cuda()
        pages = state["table"][b, :-(-(length + n) // page)].long()
        for h in range(kvheads):
            k = state["k_pages"][pages, :, h].reshape(-1, dim)[first:length + n].double()
            v = state["v_pages"][pages, :, h].reshape(-1, dim)[first:length + n].double()
            for j in range(h * group, (h + 1) * group):
                mine = slice(j * dim, (j + 1) * dim)
                q = state["q"][row:row + n, mine].double()
                score = q @ k.t() * state["scale"]
                if case["softcap"]:
                    score = torch.tanh(score / case["softcap"]) * case["softcap"]
                score = torch.where(sees, score, -math.inf)
                out[row:row + n, mine] = torch.softmax(score, -1) @ v
        row += n
    return out
