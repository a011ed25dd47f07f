"""Row operators whose permutation is data on the GPU, as programs around a language model use them.

Two permutations of that kind are in use.  A router gives every token a few experts: the tokens' rows
are sorted by expert, each expert's rows go through its own products, and the results come back,
weighted and summed (`sort`, `dispatch`, `combine`, and the gradients of the latter two).  A server keeps
the keys and values of its requests in pages: tables of pages and the slots of new tokens follow from the
requests' lengths, and rows are stored to and loaded from those slots (`tables`, `pages`).

`run` computes an operator with plain torch operations, or with this library's entry points where `own` is
true.  Rows that only move keep their bits; sums are in 32 bits and rounded once.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
MAX_BYTES = 1.2e9


def listed():
    return [
        # A decoding step of 64 requests: the router's choices as the router's top-k gives them (64-bit numbers).
        sort_case("sort_step", 64, 8, 128, 0, 128, 1, 8),
        # A batch in training or prefill, every expert's rows padded to whole tiles of a matrix product.
        sort_case("sort_batch", 32768, 8, 256, 0, 256, 64, 8),
        # A decoding step: few rows, the call itself counts.
        rows_case("dispatch_step", "dispatch", "forward", 32, 8, 128, 4096, "bf16", 1, 0.0),
        # A large batch: the largest rows written per row read.
        rows_case("dispatch_batch", "dispatch", "forward", 16384, 8, 128, 4096, "bf16", 64, 0.0),
        # Training in 32 bits at an odd token count and a width whose rows are off the 16-byte grid.
        rows_case("dispatch_grad", "dispatch", "backward", 8191, 4, 60, 2050, "f32", 16, 0.0),
        # A decoding step with six choices per token.
        rows_case("combine_step", "combine", "forward", 16, 6, 64, 5120, "f16", 1, 0.0),
        # A large batch coming back from its experts.
        rows_case("combine_batch", "combine", "forward", 16384, 8, 128, 4096, "bf16", 64, 0.0),
        # Its gradient at a training step's size, a tenth of the choices dropped by a capacity limit.
        rows_case("combine_grad", "combine", "backward", 8192, 8, 128, 4096, "bf16", 64, 0.1),
        # A decoding step: every request of a full batch gets one token.
        tables_case("tables_step", 256, 1, 8192, 16),
        # Chunked prefill: requests bring up to 2048 tokens each, some none.
        tables_case("tables_batch", 96, 2048, 32768, 64),
        # The decoding step's new keys and values into pages whose slots hold all heads.
        pages_case("store_step", "store", 256, 8, 128, "bf16", 16, "slot", 0.0),
        # All cached keys and values of a long batch, head by head, for an attention over dense tensors.
        pages_case("load_batch", "load", 131072, 8, 128, "bf16", 64, "head", 0.0),
    ]


def sort_case(name, tokens, choices, experts, first, local, align, id_bytes):
    return {"name": name, "op": "sort", "tokens": tokens, "choices": choices, "experts": experts, "first": first, "local": local,
            "align": align, "id_bytes": id_bytes}


def rows_case(name, op, direction, tokens, choices, experts, width, dtype, align, dropped):
    return {"name": name, "op": op, "direction": direction, "tokens": tokens, "choices": choices, "experts": experts, "width": width,
            "dtype": dtype, "align": align, "dropped": dropped}


def tables_case(name, requests, chunk, context, page):
    return {"name": name, "op": "tables", "requests": requests, "chunk": chunk, "context": context, "page": page}


def pages_case(name, direction, tokens, heads, width, dtype, page, layout, idle):
    return {"name": name, "op": "pages", "direction": direction, "tokens": tokens, "heads": heads, "width": width, "dtype": dtype,
            "page": page, "layout": layout, "idle": idle}


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    while True:
        op = rng.choice(["sort", "dispatch", "combine", "tables", "pages"])
        if op == "sort":
            experts = spread(8, 512)
            local = experts if rng.random() < 0.6 else max(1, experts // rng.choice([2, 4, 8]))
            case = sort_case("", spread(1, 32768), rng.randint(1, 8), experts, rng.randint(0, experts - local), local,
                             rng.choice([1, 8, 16, 64, 128]), rng.choice([4, 8]))
        elif op in ("dispatch", "combine"):
            case = rows_case("", op, rng.choice(["forward", "backward"]), spread(1, 16384), rng.randint(1, 8), spread(8, 256),
                             spread(128, 8192), rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([1, 16, 64]),
                             rng.choice([0.0, 0.0, 0.1, 0.5]))
        elif op == "tables":
            case = tables_case("", spread(1, 1024), spread(1, 2048), spread(1, 32768), rng.choice([1, 16, 32, 64, 128, 256]))
        else:
            case = pages_case("", rng.choice(["store", "load"]), spread(1, 131072), spread(1, 32), rng.choice([64, 80, 96, 128, 192, 256, 576]),
                              rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([1, 16, 64, 128]), rng.choice(["slot", "head"]),
                              rng.choice([0.0, 0.0, 0.2]))
        case.pop("name")
        case["choices"] = min(case["choices"], case["experts"]) if "choices" in case else 1
        if op in ("tables", "pages"):
            case.pop("choices")
        if work(case)["bytes"] <= MAX_BYTES:
            return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def row_bound(case):
    """Rows that hold the sorted order of any routing, which a program knows before it: every expert that gets a row may need a tile more."""
    n = case["tokens"] * case["choices"]
    return n + min(case.get("local", case["experts"]), n) * (case["align"] - 1)


def routed(case, g):
    """Distinct experts per token, some experts more in demand than others, and the choices' weights."""
    tokens, choices, experts = case["tokens"], case["choices"], case["experts"]
    demand = torch.randn(experts, generator=g, device="cuda")
    score = torch.randn(tokens, experts, generator=g, device="cuda") + demand
    top, ids = torch.topk(score, choices, dim=1)
    weights = torch.softmax(top, dim=1)
    if case.get("dropped"):
        lost = torch.rand(tokens, choices, generator=g, device="cuda") < case["dropped"]
        ids = torch.where(lost, torch.full_like(ids, -1), ids)
    return ids, weights


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op == "tables":
        return prepare_tables(case, g)
    if op == "pages":
        return prepare_pages(case, g)
    ids, weights = routed(case, g)
    tokens, choices, rows = case["tokens"], case["choices"], row_bound(case)
    if op == "sort":
        local = case["local"]
        state = {"case": case, "ids": ids if case["id_bytes"] == 8 else ids.to(torch.int32), "rows": rows}
        state["counts"] = torch.empty(local, dtype=torch.int32, device="cuda")
        state["offsets"] = torch.empty(local + 1, dtype=torch.int32, device="cuda")
        state["position"] = torch.empty(tokens, choices, dtype=torch.int32, device="cuda")
        state["source"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        if own:
            import cutt_amd as cutt
            state["workspace"] = torch.empty(cutt.cuttExpertSortWorkspace(tokens, choices, local), dtype=torch.uint8, device="cuda")
        return state
    _, _, position, source = plain_sort(ids, 0, case["experts"], case["align"], rows)
    width, dtype = case["width"], TYPES[case["dtype"]]

    def values(n):
        return torch.randn(n, width, generator=g, device="cuda", dtype=dtype)

    state = {"case": case, "position": position, "source": source, "weights": weights, "rows": rows}
    if op == "dispatch" and case["direction"] == "forward":
        state["x"] = values(tokens)
        state["y"] = torch.empty(rows, width, dtype=dtype, device="cuda")
    elif op == "dispatch":
        state["dy"] = values(rows)
        state["dx"] = torch.empty(tokens, width, dtype=dtype, device="cuda")
    elif case["direction"] == "forward":
        state["y"] = values(rows)
        state["out"] = torch.empty(tokens, width, dtype=dtype, device="cuda")
    else:
        state["y"] = values(rows)
        state["dout"] = values(tokens)
        state["dy"] = torch.empty(rows, width, dtype=dtype, device="cuda")
        state["dweights"] = torch.empty(tokens, choices, device="cuda")
    return state


def token_budget(case):
    """New tokens that a server takes into one batch: what its requests bring in the mean."""
    return case["requests"] * (case["chunk"] + 1) // 2


def prepare_tables(case, g):
    requests, page = case["requests"], case["page"]

    def whole(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    cached = whole(0, case["context"] + 1, (requests,))
    tokens = token_budget(case)
    if case["chunk"] == 1:
        added = torch.ones(requests, dtype=torch.int32, device="cuda")
    else:  # requests past the budget have to wait
        ends = torch.cumsum(whole(0, case["chunk"] + 1, (requests,)), 0).clamp(max=tokens)
        added = torch.diff(ends, prepend=ends.new_zeros(1)).to(torch.int32)
    owned = (cached + page - 1) // page
    width = (case["context"] + case["chunk"] + page - 1) // page
    pages = int(owned.sum()) + int(added.sum()) // page + requests + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")
    mine = col[None, :] < owned[:, None]
    tables[mine] = order[:int(owned.sum())]
    free = order[int(owned.sum()):].contiguous()
    return {"case": case, "cached": cached, "added": added, "free": free, "tables": tables, "tokens": tokens,
            "starts": torch.empty(requests + 1, dtype=torch.int32, device="cuda"),
            "used": torch.empty(1, dtype=torch.int32, device="cuda"),
            "slots": torch.empty(tokens, dtype=torch.int64, device="cuda"),
            "positions": torch.empty(tokens, dtype=torch.int32, device="cuda")}


def prepare_pages(case, g):
    tokens, heads, width, page, dtype = case["tokens"], case["heads"], case["width"], case["page"], TYPES[case["dtype"]]
    pages = (tokens + page - 1) // page
    pages += pages // 4 + 1  # some pages belong to nobody
    used = torch.randperm(pages, generator=g, device="cuda")[:(tokens + page - 1) // page]
    at = torch.arange(tokens, device="cuda")
    slots = used[at // page] * page + at % page
    if case["idle"]:
        slots = torch.where(torch.rand(tokens, generator=g, device="cuda") < case["idle"], torch.full_like(slots, -1), slots)
    # one page more than the requests can get, where the plain form leaves the tokens that have no slot
    shape = (pages + 1, page, heads, width) if case["layout"] == "slot" else (pages + 1, heads, page, width)
    state = {"case": case, "slots": slots, "pages": pages}
    if case["direction"] == "store":
        # keys and values lie beside the queries in the projection's output
        qkv = torch.randn(tokens, 4 * heads, width, generator=g, device="cuda", dtype=dtype)
        state["k"], state["v"] = qkv[:, 2 * heads:3 * heads], qkv[:, 3 * heads:]
        state["k_cache"] = torch.zeros(shape, dtype=dtype, device="cuda")
        state["v_cache"] = torch.zeros(shape, dtype=dtype, device="cuda")
    else:
        state["k_cache"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
        state["v_cache"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
        state["k"] = torch.empty(heads, tokens, width, dtype=dtype, device="cuda")
        state["v"] = torch.empty(heads, tokens, width, dtype=dtype, device="cuda")
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return {"sort": own_sort, "dispatch": own_dispatch, "combine": own_combine, "tables": own_tables, "pages": own_pages}[op](state)
    if op == "sort":
        counts, offsets, position, source = plain_sort(state["ids"], case["first"], case["local"], case["align"], state["rows"])
        return {"counts": counts, "offsets": offsets, "position": position, "source": source}
    if op == "tables":
        return plain_tables(state)
    if op == "pages":
        return plain_pages(state)
    if op == "dispatch":
        if case["direction"] == "forward":
            token = torch.div(state["source"], case["choices"], rounding_mode="floor").clamp(min=0)
            return state["x"][token].masked_fill_((state["source"] < 0)[:, None], 0)
        return plain_sum(state["dy"], state["position"], None)
    if case["direction"] == "forward":
        return plain_sum(state["y"], state["position"], state["weights"])
    return plain_combine_backward(state)


def plain_sort(ids, first, experts, align, rows):
    shape = ids.shape
    key = ids.reshape(-1).long() - first
    key = torch.where((key >= 0) & (key < experts), key, experts)
    n = key.numel()
    order = torch.argsort(key, stable=True)
    expert = key[order]
    count = torch.zeros(experts + 1, dtype=torch.int64, device=key.device).scatter_add_(0, key, torch.ones_like(key))
    padded = (count[:experts] + align - 1) // align * align
    offsets = torch.cat([padded.new_zeros(1), torch.cumsum(padded, 0)])
    rank = torch.arange(n, device=key.device) - (torch.cumsum(count, 0) - count)[expert]
    row = offsets[expert] + rank
    row = torch.where((expert < experts) & (row < rows), row, -1)
    position = torch.empty_like(row)
    position[order] = row
    source = torch.full((rows + 1,), -1, dtype=torch.int32, device=key.device)
    source[torch.where(row >= 0, row, rows)] = order.int()
    return count[:experts].int(), offsets.int(), position.int().reshape(shape), source[:rows]


def plain_sum(y, position, weights):
    out = torch.zeros(position.shape[0], y.shape[1], device=y.device)
    for k in range(position.shape[1]):
        there = position[:, k] >= 0
        row = y[position[:, k].clamp(min=0)].float()
        if weights is not None:
            row = row * weights[:, k:k + 1]
        out += torch.where(there[:, None], row, 0.0)
    return out.to(y.dtype)


def plain_combine_backward(state):
    position, source, weights, y, dout = state["position"], state["source"], state["weights"], state["y"], state["dout"]
    choices = position.shape[1]
    from_choice = source.clamp(min=0)
    token = torch.div(from_choice, choices, rounding_mode="floor")
    scale = torch.where(source >= 0, weights.reshape(-1)[from_choice], 0.0)
    dy = (dout[token].float() * scale[:, None]).masked_fill_((source < 0)[:, None], 0.0).to(y.dtype)
    dweights = torch.empty_like(weights)
    grad = dout.float()
    for k in range(choices):
        dot = (grad * y[position[:, k].clamp(min=0)].float()).sum(1)
        dweights[:, k] = torch.where(position[:, k] >= 0, dot, 0.0)
    return {"dy": dy, "dweights": dweights}


def plain_tables(state):
    page = state["case"]["page"]
    cached, added, free, tables = state["cached"].long(), state["added"].long(), state["free"], state["tables"]
    width = tables.shape[1]
    owned = (cached + page - 1) // page
    want = (cached + added + page - 1) // page
    need = want - owned
    first = torch.cumsum(need, 0) - need
    starts = torch.cat([added.new_zeros(1), torch.cumsum(added, 0)])
    col = torch.arange(width, device=tables.device)[None, :]
    fresh = (col >= owned[:, None]) & (col < want[:, None])
    at = first[:, None] + col - owned[:, None]
    taken = torch.where(at < free.numel(), free[at.clamp(0, max(free.numel() - 1, 0))], -1)
    tables = torch.where(fresh, taken, tables)
    i = torch.arange(state["tokens"], device=tables.device)
    b = torch.searchsorted(starts[1:], i, right=True)
    there = b < cached.numel()
    b = b.clamp(max=cached.numel() - 1)
    pos = cached[b] + i - starts[b]
    slot_page = tables[b, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(there & (slot_page >= 0), slot_page * page + pos % page, -1)
    return {"tables": tables, "starts": starts.int(), "used": need.sum().int().reshape(1), "slots": slots,
            "positions": torch.where(there, pos, -1).int()}


def plain_pages(state):
    case, slots = state["case"], state["slots"]
    page = case["page"]
    there = slots >= 0
    at = torch.where(there, torch.div(slots, page, rounding_mode="floor"), state["pages"])
    off = torch.where(there, slots % page, 0)
    if case["direction"] == "store":
        for rows, cache in ((state["k"], state["k_cache"]), (state["v"], state["v_cache"])):
            if case["layout"] == "slot":
                cache[at, off] = rows
            else:
                cache[at, :, off] = rows
        return {"k_cache": state["k_cache"][:state["pages"]], "v_cache": state["v_cache"][:state["pages"]]}
    out = {}
    for name in ("k", "v"):
        cache = state[name + "_cache"]
        rows = cache[at, off] if case["layout"] == "slot" else cache[at, :, off]
        out[name] = rows.masked_fill_(~there[:, None, None], 0).transpose(0, 1).contiguous()
    return out


# ---------------------------------------------------------------------------
# the same through this library
# ---------------------------------------------------------------------------
def checked(code, what):
    if code:
        import cutt_amd as cutt
        raise cutt.CuttError(code, what)


def stream():
    return torch.cuda.current_stream().cuda_stream


def own_sort(state):
    import cutt_amd as cutt
    case, space = state["case"], state["workspace"]
    checked(cutt.cuttExpertSort(case["tokens"], case["choices"], case["first"], case["local"], case["align"], state["rows"], case["id_bytes"], stream(),
                                state["ids"].data_ptr(), state["counts"].data_ptr(), state["offsets"].data_ptr(), state["position"].data_ptr(),
                                state["source"].data_ptr(), space.data_ptr(), space.numel()), "cuttExpertSort")
    return {"counts": state["counts"], "offsets": state["offsets"], "position": state["position"], "source": state["source"]}


def row_type(case):
    import cutt_amd as cutt
    return {"f32": cutt.CUTT_F32, "f16": cutt.CUTT_F16, "bf16": cutt.CUTT_BF16}[case["dtype"]]


def own_dispatch(state):
    import cutt_amd as cutt
    case, width = state["case"], state["case"]["width"]
    if case["direction"] == "forward":
        checked(cutt.cuttExpertDispatch(case["tokens"], case["choices"], state["rows"], width, SIZES[case["dtype"]], stream(), state["position"].data_ptr(),
                                        state["source"].data_ptr(), state["x"].data_ptr(), width, state["y"].data_ptr(), width), "cuttExpertDispatch")
        return state["y"]
    checked(cutt.cuttExpertDispatchBackward(case["tokens"], case["choices"], state["rows"], width, row_type(case), stream(), state["position"].data_ptr(),
                                            state["dy"].data_ptr(), width, state["dx"].data_ptr(), width), "cuttExpertDispatchBackward")
    return state["dx"]


def own_combine(state):
    import cutt_amd as cutt
    case, width = state["case"], state["case"]["width"]
    if case["direction"] == "forward":
        checked(cutt.cuttExpertCombine(case["tokens"], case["choices"], state["rows"], width, row_type(case), stream(), state["position"].data_ptr(),
                                       state["weights"].data_ptr(), state["y"].data_ptr(), width, state["out"].data_ptr(), width), "cuttExpertCombine")
        return state["out"]
    checked(cutt.cuttExpertCombineBackward(case["tokens"], case["choices"], state["rows"], width, row_type(case), stream(), state["position"].data_ptr(),
                                           state["source"].data_ptr(), state["weights"].data_ptr(), state["y"].data_ptr(), width,
                                           state["dout"].data_ptr(), width, state["dy"].data_ptr(), width, state["dweights"].data_ptr()),
            "cuttExpertCombineBackward")
    return {"dy": state["dy"], "dweights": state["dweights"]}


def own_tables(state):
    import cutt_amd as cutt
    case, tables = state["case"], state["tables"]
    checked(cutt.cuttPageTables(case["requests"], case["page"], tables.shape[1], state["free"].numel(), state["tokens"], stream(), state["cached"].data_ptr(),
                                state["added"].data_ptr(), state["free"].data_ptr(), tables.data_ptr(), state["starts"].data_ptr(),
                                state["used"].data_ptr(), state["slots"].data_ptr(), state["positions"].data_ptr()), "cuttPageTables")
    return {name: state[name] for name in ("tables", "starts", "used", "slots", "positions")}


def own_pages(state):
    import cutt_amd as cutt
    case, k, k_cache = state["case"], state["k"], state["k_cache"]
    store = case["direction"] == "store"
    # strides in elements: of a token and a head; of a page, a slot in it and a head
    rows = (k.stride(0), k.stride(1)) if store else (k.stride(1), k.stride(0))
    if case["layout"] == "slot":
        cache = (k_cache.stride(0), k_cache.stride(1), k_cache.stride(2))
    else:
        cache = (k_cache.stride(0), k_cache.stride(2), k_cache.stride(1))
    call = cutt.cuttPageStore if store else cutt.cuttPageLoad
    checked(call(case["tokens"], case["heads"], case["width"], SIZES[case["dtype"]], state["pages"], case["page"], stream(), state["slots"].data_ptr(),
                 k.data_ptr(), state["v"].data_ptr(), rows, k_cache.data_ptr(), state["v_cache"].data_ptr(), cache),
            "cuttPageStore" if store else "cuttPageLoad")
    if store:
        return {"k_cache": k_cache[:state["pages"]], "v_cache": state["v_cache"][:state["pages"]]}
    return {"k": k, "v": state["v"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and what it has to give
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "sort":
        n = case["tokens"] * case["choices"]
        return {"bytes": n * (case["id_bytes"] + 4) + 4 * row_bound(case) + 4 * (2 * case["local"] + 1), "flops": n}
    if op == "tables":
        tokens = token_budget(case)
        fresh = tokens / case["page"]
        return {"bytes": int(12 * tokens + 8 * fresh + 4 * (3 * case["requests"] + 2)), "flops": int(4 * tokens)}
    if op == "pages":
        tokens = case["tokens"] * (1.0 - case["idle"])
        rows = 2 * case["heads"] * case["width"] * SIZES[case["dtype"]]
        written = tokens if case["direction"] == "store" else case["tokens"]
        return {"bytes": int(8 * case["tokens"] + (tokens + written) * rows), "flops": 0}
    kept = case["tokens"] * case["choices"] * (1.0 - case["dropped"])
    n = case["tokens"] * case["choices"]
    rows = row_bound(case)
    row = case["width"] * SIZES[case["dtype"]]
    if op == "dispatch" and case["direction"] == "forward":
        return {"bytes": int(case["tokens"] * row + rows * (row + 4) + 4 * n), "flops": 0}
    if op == "dispatch":
        return {"bytes": int(kept * row + 4 * n + case["tokens"] * row), "flops": int(kept * case["width"])}
    if case["direction"] == "forward":
        return {"bytes": int(kept * row + 8 * n + case["tokens"] * row), "flops": int(2 * kept * case["width"])}
    return {"bytes": int((kept + rows + case["tokens"]) * row + 12 * n + 4 * rows), "flops": int(3 * kept * case["width"])}


def exact(case, seed):
    """The floating outputs in 64 bits, from the rows' destinations where the plain form goes by their sources and the other way round."""
    op = case["op"]
    if op in ("sort", "tables"):
        return None
    state = prepare(case, seed)
    if op == "pages":
        return exact_pages(case, state)
    position, rows, width = state["position"].long(), state["rows"], case["width"]
    tokens = case["tokens"]
    held = (state["source"] >= 0).nonzero()[:, 0]
    choice = state["source"][held].long()
    token = torch.div(choice, case["choices"], rounding_mode="floor")
    weight = state["weights"].double().reshape(-1)[choice]
    if case["direction"] == "forward" and op == "dispatch":
        y = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
        for k in range(case["choices"]):
            there = (position[:, k] >= 0).nonzero()[:, 0]
            y[position[there, k]] = state["x"][there].double()
        return y
    if op == "dispatch" or case["direction"] == "forward":
        rows_in = state["dy"] if op == "dispatch" else state["y"]
        out = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
        for lo in range(0, held.numel(), 16384):
            part = rows_in[held[lo:lo + 16384]].double()
            if op == "combine":
                part *= weight[lo:lo + 16384, None]
            out.index_add_(0, token[lo:lo + 16384], part)
        return out
    dy = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    dweights = torch.zeros(tokens * case["choices"], dtype=torch.float64, device="cuda")
    for lo in range(0, held.numel(), 16384):
        at = held[lo:lo + 16384]
        grad = state["dout"][token[lo:lo + 16384]].double()
        dy[at] = grad * weight[lo:lo + 16384, None]
        dweights[choice[lo:lo + 16384]] = (grad * state["y"][at].double()).sum(1)
    return {"dy": dy, "dweights": dweights.reshape(tokens, case["choices"])}


def exact_pages(case, state):
    pages, page, heads, width = state["pages"], case["page"], case["heads"], case["width"]
    out = {}
    for name in ("k", "v"):
        cache = state[name + "_cache"][:pages]
        flat = (cache if case["layout"] == "slot" else cache.transpose(1, 2)).reshape(pages * page, heads, width).double()
        there = (state["slots"] >= 0).nonzero()[:, 0]
        if case["direction"] == "store":
            flat[state["slots"][there]] = state[name][there].double()
            whole = flat.reshape(pages, page, heads, width)
            out[name + "_cache"] = whole if case["layout"] == "slot" else whole.transpose(1, 2).contiguous()
        else:
            rows = torch.zeros(heads, case["tokens"], width, dtype=torch.float64, device="cuda")
            rows[:, there] = flat[state["slots"][there]].transpose(0, 1)
            out[name] = rows
    return out
