"""Timing cases of batched serving over a paged KV cache.

Each case is a plain dict; `kind` names the call that a program makes in a step
of a batch of requests:

  step    Context.page_step: block tables, slot map, positions and newest rows
          of the step, from the requests' lengths and their new tokens
  append  the step's rows into the pages: HeadTransform.append_paged (raw
          projections through the head norms and the rotation at each row's own
          position) where `transform` is set, else Context.paged_append
  attend  Context.paged_attention: the newest token of every request over its
          pages

`run` makes these calls where `own` is set and computes the same from elementary
torch operations where it is not. The heads are those of the attention cases
beside this file (16 query and 8 KV heads of 256 dims, sliding layers with a
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
EPSILON = 1e-6
ROPE_BASE = 10000.0
SLIDING = (16, 8, 256)
GLOBAL = (16, 2, 512)
SPARE_PAGES = 5
_contexts = {}


# ---- cases ------------------------------------------------------------------

def _step(requests, longest, page, prompts=0, prompt=0, idle=0):
    return {"kind": "step", "requests": requests, "longest": longest, "page": page,
            "prompts": prompts, "prompt": prompt, "idle": idle}


def _append(heads, rows, run, longest, page, dtype, transform):
    qheads, kvheads, dim = heads
    return {"kind": "append", "qheads": qheads, "kvheads": kvheads, "dim": dim, "rows": rows,
            "run": run, "longest": longest, "page": page, "dtype": dtype, "transform": transform}


def _attend(heads, requests, shortest, longest, page, dtype, window=0, idle=0, softcap=0.0):
    qheads, kvheads, dim = heads
    return {"kind": "attend", "qheads": qheads, "kvheads": kvheads, "dim": dim,
            "requests": requests, "shortest": shortest, "longest": longest, "page": page,
            "dtype": dtype, "window": window, "idle": idle, "softcap": softcap}


def listed():
    return [
        # a small batch's decode step: one token each, launch latency counts
        {"name": "step_decode_64", **_step(64, 8192, 16)},
        # a busy server's step: decoding requests, some idle slots of the
        # batch, and a few prompts let in beside them
        {"name": "step_mixed_512", **_step(512, 8192, 16, prompts=6, prompt=2000, idle=37)},
        # a batch of prompts alone, small pages: many slots and new pages
        {"name": "step_prompts_96", **_step(96, 1, 16, prompts=96, prompt=4096)},
        # one decode token of 64 requests through the head transform
        {"name": "append_decode_64",
         **_append(SLIDING, 64, 1, 8192, 16, "f32", True)},
        # prompts of 500 tokens through the head transform into bf16 pages
        {"name": "append_prompts_6000",
         **_append(SLIDING, 6000, 500, 2000, 32, "bf16", True)},
        # prepared rows of a global layer's prompt moved into f32 pages as
        # they are
        {"name": "append_rows_3001_d512",
         **_append(GLOBAL, 3001, 3001, 4000, 64, "f32", False)},
        # one young conversation: every part of the latency shows
        {"name": "attend_1x100", **_attend(SLIDING, 1, 100, 100, 16, "f32")},
        # a batch of conversations of very different lengths, two of its slots
        # idle
        {"name": "attend_64x8k_bf16", **_attend(SLIDING, 64, 64, 8192, 16, "bf16", idle=2)},
        # a sliding layer of long conversations: the window starts inside
        # pages and key chunks
        {"name": "attend_32_window", **_attend(SLIDING, 32, 2000, 16384, 16, "f32", window=1024)},
        # a global layer of long conversations, the most bytes
        {"name": "attend_16x32k_d512", **_attend(GLOBAL, 16, 2048, 32768, 64, "f32")},
        # one very long document in bf16 pages
        {"name": "attend_1x128k_d512_bf16", **_attend(GLOBAL, 1, 131072, 131072, 64, "bf16")},
        # many short chats, four query heads to a KV head
        {"name": "attend_256x2k_d128_bf16",
         **_attend((32, 8, 128), 256, 16, 2048, 16, "bf16", idle=7)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = (SLIDING, SLIDING, GLOBAL, (32, 8, 128), (16, 4, 64), (10, 2, 80), (32, 1, 128))
TRANSFORM_HEADS = (SLIDING, SLIDING, GLOBAL, (32, 8, 128), (16, 4, 64))


def draw(rng):
    """One more case: sizes over the logarithm of each range."""
    while True:
        kind = rng.choice(("step", "append", "attend", "attend"))
        page = rng.choice((8, 16, 16, 32, 48, 64, 128))
        dtype = rng.choice(("f32", "bf16"))
        if kind == "step":
            requests = _log(rng, 1, 1024)
            prompts = rng.choice((0, min(requests, _log(rng, 1, 64))))
            idle = rng.choice((0, (requests - prompts) // 7))
            case = _step(requests, _log(rng, 16, 16384), page, prompts, _log(rng, 16, 4096), idle)
            if prompts * case["prompt"] > 300000 or requests * case["longest"] > 1 << 22:
                continue
        elif kind == "append":
            transform = rng.choice((True, True, False))
            heads = rng.choice(TRANSFORM_HEADS if transform else HEADS)
            run = rng.choice((1, 1, _log(rng, 2, 4096)))
            requests = _log(rng, 1, 256)
            case = _append(heads, requests * run, run, _log(rng, 4200, 16384), page, dtype,
                           transform)
            if case["rows"] > 6000:
                continue
        else:
            heads = rng.choice(HEADS)
            requests = _log(rng, 1, 256)
            longest = _log(rng, 16, 65536)
            case = _attend(heads, requests, max(1, longest // rng.choice((1, 4, 64))), longest,
                           page, dtype, window=rng.choice((0, 0, 0, 1024)),
                           idle=rng.choice((0, requests // 9)),
                           softcap=rng.choice((0.0, 0.0, 0.0, 50.0)))
            if requests * longest * heads[1] * heads[2] > 1 << 29 or work(case)["bytes"] > 1.7e9:
                continue
        return case


# ---- a case's lengths (the same for every seed) -----------------------------

def _spread(n, low, high):
    """n lengths spread over the logarithm of [low, high], high among them."""
    i = np.arange(n)
    x = np.round(low * (high / low) ** ((0.6180339887498949 * i + 0.37) % 1.0)).astype(np.int64)
    if n:
        x[n // 2] = high
    return x


def _step_lengths(case):
    """(lengths, counts): prompts first, idle requests last."""
    b, prompts, idle = case["requests"], case["prompts"], case["idle"]
    lengths = np.zeros(b, np.int64)
    counts = np.ones(b, np.int64)
    lengths[prompts:] = _spread(b - prompts, 1, case["longest"])
    if prompts:
        counts[:prompts] = _spread(prompts, max(1, case["prompt"] // 16), case["prompt"])
    if idle:
        counts[b - idle:] = 0
    return lengths, counts


def _append_positions(case):
    """(request, position) of every row: runs of consecutive tokens."""
    n, run = case["rows"], case["run"]
    request = np.arange(n) // run
    first = _spread(request[-1] + 1, 1, max(1, case["longest"] - run)) if n else np.zeros(0)
    return request, first[request] + np.arange(n) % run


def _attend_lengths(case):
    """(lengths, rows): idle requests have no row, every third of them no keys."""
    b, idle = case["requests"], case["idle"]
    lengths = _spread(b, case["shortest"], case["longest"])
    rows = np.full(b, -1, np.int64)
    # idle slots lie among the others
    off = np.zeros(b, bool)
    if idle:
        off[np.arange(idle) * (b // idle)] = True
        lengths[np.flatnonzero(off)[::3]] = 0
    rows[~off] = np.arange(int((~off).sum()))
    return lengths, rows


def _pages(lengths, page):
    return -(-np.asarray(lengths) // page)


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
    if case["kind"] == "step":
        _prepare_step(state, rng)
    elif case["kind"] == "append":
        _prepare_append(state, rng, randn)
    else:
        _prepare_attend(state, rng, randn)
    return state


def _prepare_step(state, rng):
    case = state["case"]
    page = case["page"]
    lengths, counts = _step_lengths(case)
    stride = int(_pages(lengths + counts, page).max()) + 3
    new = int((_pages(lengths + counts, page) - _pages(lengths, page)).sum())
    table, free = _table(lengths, stride, page, rng, new + SPARE_PAGES)
    pages = int(_pages(lengths, page).sum()) + new + SPARE_PAGES
    free_pages = np.full(pages, -1, np.int32)
    free_pages[:len(free)] = free
    # a captured step has room for more rows than most steps use
    rows = int(counts.sum()) + 11
    state.update(pages=pages, rows=rows, stride=stride,
                 lengths=_ints(lengths), counts=_ints(counts), table=_ints(table),
                 free_pages=_ints(free_pages), counters=_ints([len(free), 0, 0, 0]))
    for name, n in (("step_lengths", case["requests"]), ("newest", case["requests"]),
                    ("slots", rows), ("positions", rows), ("row_request", rows)):
        state[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
    if own:
        names = ("lengths", "table", "free_pages", "counters", "step_lengths", "newest", "slots",
                 "positions", "row_request")
        state["batch"] = _package().page_batch(
            requests=case["requests"], table_stride=stride, page_tokens=page, pages=pages,
            step_rows=rows, **{n: state[n].data_ptr() for n in names})


def _prepare_append(state, rng, randn):
    case = state["case"]
    page, kvheads, dim = case["page"], case["kvheads"], case["dim"]
    request, position = _append_positions(case)
    n = case["rows"]
    padded = n + 3  # the last rows of the step have no token
    key = request.astype(np.int64) << 32 | position // page
    _, which = np.unique(key, return_inverse=True)
    pages = int(which.max()) + 1 + SPARE_PAGES
    order = rng.permutation(pages)
    slots = np.full(padded, -1, np.int64)
    slots[:n] = order[which] * page + position % page
    positions = np.full(padded, -1, np.int64)
    positions[:n] = position
    dtype = _types(case["dtype"])
    state.update(pages=pages, rows=padded, slots=_ints(slots), positions=_ints(positions),
                 k_pages=randn(pages, page, kvheads, dim, dtype=dtype),
                 v_pages=randn(pages, page, kvheads, dim, dtype=dtype),
                 keys=randn(padded, kvheads, dim), values=randn(padded, kvheads, dim))
    if case["transform"]:
        state.update(queries=randn(padded, case["qheads"], dim),
                     q_out=torch.zeros(padded, case["qheads"], dim, device="cuda"),
                     q_scale=1.0 + 0.1 * randn(dim), k_scale=1.0 + 0.1 * randn(dim),
                     frequencies=torch.from_numpy(_frequencies(dim)).cuda())
    if own:
        pcl = _package()
        state["pools"] = _pools(state)
        if case["transform"]:
            state["transform"] = pcl.HeadTransform(
                _context(), case["qheads"], kvheads, dim, state["q_scale"].cpu().numpy(),
                state["k_scale"].cpu().numpy(), EPSILON, ROPE_BASE)


def _prepare_attend(state, rng, randn):
    case = state["case"]
    page, qheads, kvheads, dim = case["page"], case["qheads"], case["kvheads"], case["dim"]
    lengths, rows = _attend_lengths(case)
    stride = int(_pages(case["longest"], page)) + 2
    table, _ = _table(lengths, stride, page, rng, SPARE_PAGES)
    pages = int(_pages(lengths, page).sum()) + SPARE_PAGES
    n = case["requests"]
    dtype = _types(case["dtype"])
    state.update(pages=pages, stride=stride, scale=float(np.float32(1.0 / math.sqrt(dim))),
                 lengths=_ints(lengths), rows=_ints(rows), table=_ints(table),
                 k_pages=randn(pages, page, kvheads, dim, dtype=dtype),
                 v_pages=randn(pages, page, kvheads, dim, dtype=dtype),
                 q=randn(n, qheads * dim), out=torch.zeros(n + 1, qheads * dim, device="cuda"))
    if own:
        context = _context()
        state["desc"] = context.paged_desc(
            pools=_pools(state), q=state["q"].data_ptr(), q_stride=qheads * dim, q_rows=n,
            qheads=qheads, table=state["table"].data_ptr(), table_stride=stride,
            lengths=state["lengths"].data_ptr(), rows=state["rows"].data_ptr(), requests=n,
            max_length=case["longest"], window=case["window"], q_scale=state["scale"],
            softcap=case["softcap"], out=state["out"].data_ptr(), o_stride=qheads * dim)
        context.reserve(context.paged_workspace_bytes(state["desc"]))


def _pools(state):
    case = state["case"]
    pcl = _package()
    return pcl.page_pools(
        k=state["k_pages"].data_ptr(), v=state["v_pages"].data_ptr(),
        type=pcl.CACHE_F32 if case["dtype"] == "f32" else pcl.CACHE_BF16, pages=state["pages"],
        page_tokens=case["page"], kvheads=case["kvheads"], dim=case["dim"])


# ---- one pass ---------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "step":
        return _run_step(state)
    if kind == "append":
        return _run_append(state)
    return _run_attend(state)


def _run_step(state):
    if own:
        _context().page_step(state["batch"], state["counts"].data_ptr())
        return [state[n] for n in ("slots", "positions", "row_request", "step_lengths", "newest",
                                   "table")] + [state["counters"][:3]]
    case = state["case"]
    page = case["page"]
    lengths, counts = state["lengths"].long(), state["counts"].long()
    after = lengths + counts
    held = (lengths + page - 1) // page
    need = (after + page - 1) // page - held
    row_end, page_end = counts.cumsum(0), need.cumsum(0)
    free = state["counters"][0].long()
    # new pages of a request from the top of the free list, in request order
    column = torch.arange(state["stride"], device="cuda")
    taken = (page_end - need)[:, None] + column - held[:, None]
    new = (column >= held[:, None]) & (column < (held + need)[:, None])
    picked = state["free_pages"][torch.where(new, free - 1 - taken, 0)]
    table = torch.where(new, picked, state["table"])
    # rows of the step
    row = torch.arange(state["rows"], device="cuda")
    inside = row < row_end[-1]
    request = torch.searchsorted(row_end, row, right=True).clamp(max=case["requests"] - 1)
    position = lengths[request] + row - (row_end - counts)[request]
    slot = table[request, (position // page).clamp(max=state["stride"] - 1)].long() * page \
        + position % page
    out = [torch.where(inside, x, -1).int() for x in (slot, position, request)]
    newest = torch.where(counts > 0, row_end - 1, -1).int()
    counters = torch.stack((free, row_end[-1], page_end[-1])).int()
    return out + [after.int(), newest, table, counters]


def _frequencies(dim):
    """1 / base^(2j/dim) in f32, as the rotation's definition has them."""
    exponent = 2 * np.arange(dim // 2, dtype=np.float32) / np.float32(dim)
    power = np.power(np.float64(ROPE_BASE), exponent.astype(np.float64)).astype(np.float32)
    return np.float32(1.0) / power


def _transformed(x, scale, angle, wide):
    """Head norm over the last axis, the learned scale, then the rotation of
    pairs (j, j + dim/2) by the rows' angles; neither for values."""
    y = x.to(wide)
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPSILON)
    if scale is None:
        return y
    y = y * scale.to(wide)
    half = x.shape[-1] // 2
    s, c = (f(angle.double()).to(wide)[:, None, :] for f in (torch.sin, torch.cos))
    a, b = y[..., :half], y[..., half:]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _place(pages, slots, rows):
    """Rows into their slots; a row without a slot repeats the first row."""
    flat = pages.view(-1, *pages.shape[2:])
    inside = slots >= 0
    at = torch.where(inside, slots, slots[0]).long()
    flat[at] = torch.where(inside[:, None, None], rows, rows[:1]).to(pages.dtype)


def _run_append(state):
    case = state["case"]
    if own:
        n = state["rows"]
        if case["transform"]:
            state["transform"].append_paged(
                state["pools"], state["slots"].data_ptr(), state["positions"].data_ptr(),
                case["longest"], state["queries"].data_ptr(), state["keys"].data_ptr(),
                state["values"].data_ptr(), n, state["q_out"].data_ptr())
        else:
            _context().paged_append(state["pools"], state["slots"].data_ptr(),
                                    state["keys"].data_ptr(), state["values"].data_ptr(), n)
    elif case["transform"]:
        slots = state["slots"]
        angle = state["positions"].float()[:, None] * state["frequencies"]
        _place(state["k_pages"], slots,
               _transformed(state["keys"], state["k_scale"], angle, torch.float32))
        _place(state["v_pages"], slots, _transformed(state["values"], None, None, torch.float32))
        q = _transformed(state["queries"], state["q_scale"], angle, torch.float32)
        state["q_out"].copy_(torch.where((slots >= 0)[:, None, None], q, state["q_out"]))
    else:
        _place(state["k_pages"], state["slots"], state["keys"])
        _place(state["v_pages"], state["slots"], state["values"])
    pages = [state["k_pages"], state["v_pages"]]
    return [state["q_out"]] + pages if case["transform"] else pages


def _run_attend(state):
    case = state["case"]
    if own:
        _context().paged_attention(state["desc"])
        return state["out"][:-1]
    page, qheads, kvheads, dim = case["page"], case["qheads"], case["kvheads"], case["dim"]
    n, window = case["requests"], case["window"]
    span = min(window, case["longest"]) if window else case["longest"]
    lengths, rows = state["lengths"].long(), state["rows"].long()
    key = (lengths - span).clamp(min=0)[:, None] + torch.arange(span, device="cuda")
    inside = key < lengths[:, None]
    key = torch.where(inside, key, 0)
    slot = state["table"].gather(1, key // page).clamp(min=0).long() * page + key % page
    q = state["q"][rows.clamp(min=0)].view(n, kvheads, qheads // kvheads, dim) * state["scale"]
    k = state["k_pages"].view(-1, kvheads, dim)[slot].float().permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(q, k)
    del k
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    score = score.masked_fill(~inside[:, None, None, :], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    v = state["v_pages"].view(-1, kvheads, dim)[slot].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(weight, v) / weight.sum(-1, keepdim=True)
    # requests without a row write the row behind the last
    state["out"][torch.where(rows < 0, n, rows)] = out.view(n, qheads * dim)
    return state["out"][:-1]


# ---- what a pass cannot do without, and its result in 64 bits ---------------

def work(case):
    if case["kind"] == "step":
        lengths, counts = _step_lengths(case)
        page = case["page"]
        rows = int(counts.sum())
        new = int((_pages(lengths + counts, page) - _pages(lengths, page)).sum())
        # lengths and counts read; lengths and newest rows written; a new
        # page's word read and written; three words a row written
        return {"bytes": 16 * case["requests"] + 8 * new + 12 * (rows + 11), "flops": 8 * rows}
    size = 4 if case["dtype"] == "f32" else 2
    width = case["kvheads"] * case["dim"]
    if case["kind"] == "append":
        n = case["rows"]
        total = n * (2 * width * (4 + size) + 4)
        flops = 0
        if case["transform"]:
            q = case["qheads"] * case["dim"]
            total += n * (8 * q + 4 + 4 * case["dim"])
            flops = n * (8 * (q + width) + 4 * width)
        return {"bytes": total, "flops": flops}
    lengths, rows = _attend_lengths(case)
    active = rows >= 0
    keys = lengths[active]
    if case["window"]:
        keys = np.minimum(keys, case["window"])
    q = case["qheads"] * case["dim"]
    total = int(keys.sum())
    return {"bytes": 2 * size * width * total + 4 * int(_pages(keys, case["page"]).sum())
            + 8 * q * int(active.sum()) + 8 * case["requests"], "flops": 4 * q * total}


def exact(case, seed):
    if case["kind"] == "step":
        return None
    state = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(state)
    return _exact_attend(state)


def _exact_append(state):
    case = state["case"]
    slots = state["slots"].cpu().numpy()
    used = np.flatnonzero(slots >= 0)
    at = torch.from_numpy(slots[used].astype(np.int64)).cuda()
    rows = torch.from_numpy(used).cuda()

    def norm(x):
        x = x.double()
        return x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPSILON)

    def rotate(x, scale):
        # the angle is an f32 by definition
        angle = (state["positions"][rows].float()[:, None] * state["frequencies"]).double()
        x = norm(x) * scale.double()
        a, b = x.chunk(2, -1)
        s, c = torch.sin(angle)[:, None], torch.cos(angle)[:, None]
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    keys, values = state["keys"][rows], state["values"][rows]
    out = []
    if case["transform"]:
        q = torch.zeros(state["q_out"].shape, dtype=torch.float64, device="cuda")
        q[rows] = rotate(state["queries"][rows], state["q_scale"])
        out.append(q)
        keys, values = rotate(keys, state["k_scale"]), norm(values)
    for pages, new in ((state["k_pages"], keys), (state["v_pages"], values)):
        wide = pages.double()
        wide.view(-1, case["kvheads"], case["dim"])[at] = new.double()
        out.append(wide)
    return out


def _exact_attend(state):
    case = state["case"]
    page, qheads, kvheads, dim = case["page"], case["qheads"], case["kvheads"], case["dim"]
    group = qheads // kvheads
    out = torch.zeros(case["requests"], qheads * dim, dtype=torch.float64, device="cuda")
    lengths, rows = state["lengths"].tolist(), state["rows"].tolist()
    for i, (length, row) in enumerate(zip(lengths, rows)):
        if row < 0:
            continue
        first = max(0, length - case["window"]) if case["window"] else 0
        pages = state["table"][i, :-(-length // page)].long()
        for h in range(kvheads):
            k = state["k_pages"][pages, :, h].reshape(-1, dim)[first:length].double()
            v = state["v_pages"][pages, :, h].reshape(-1, dim)[first:length].double()
            q = state["q"][row].view(qheads, dim)[h * group:(h + 1) * group].double()
            score = q @ k.t() * state["scale"]
            if case["softcap"]:
                score = torch.tanh(score / case["softcap"]) * case["softcap"]
            out[row].view(qheads, dim)[h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out
