"""Products on rows that the row operators lay out, as programs around a language model use them.

Experts' products: rows sorted by expert lie in ragged segments, and every segment is multiplied by its expert's weights
(`product`; with the weights transposed it is the gradient for the rows too); the weights' gradient sums over a segment's rows
(`weights`).  Attention over pages: new tokens' queries see the keys and values of their requests' earlier tokens, which lie in
pages (`attend`): one query per request and step, or a few where tokens were drafted ahead.

`run` computes an operator with plain torch operations, or with this library's entry points where `own` is true.  Sums are in 32
bits and rounded once.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
MAX_BYTES = 1.7e9
MAX_FLOPS = {"f32": 1.5e11, "f16": 1.6e12, "bf16": 1.6e12}


def listed():
    return [
        # A decoding step of a small model: a handful of rows, the call itself counts.
        product_case("product_few", "product", 4, 2, 8, 1024, 512, "f16", True, 1),
        # A decoding step of 64 requests: a few rows per expert, every expert's weights are read.
        product_case("product_step", "product", 64, 8, 128, 4096, 1536, "bf16", False, 1),
        # A chunk of a prompt: about 64 rows per expert.
        product_case("product_chunk", "product", 512, 8, 64, 2048, 1408, "f16", True, 16),
        # A large batch in training or prefill.
        product_case("product_batch", "product", 16384, 8, 128, 4096, 1536, "bf16", False, 16),
        # Training in 32 bits: the gradient for the rows, at an odd token count and widths off the 16-byte grid.
        product_case("product_odd", "product", 2047, 4, 60, 690, 2050, "f32", True, 1),
        # The weights' gradient of a training step.
        product_case("weights_batch", "weights", 8192, 8, 64, 4096, 1536, "bf16", False, 16),
        # The same of a small batch: short segments, some of them empty.
        product_case("weights_chunk", "weights", 100, 2, 64, 1000, 520, "f16", False, 1),
        # In 32 bits, off the grid.
        product_case("weights_odd", "weights", 2047, 4, 60, 2050, 690, "f32", False, 1),
        # A decoding step of a few requests.
        attend_case("attend_few", 8, 1, 2048, "ragged", 0, 32, 8, 128, "bf16", 16, "slot", 0.0),
        # A full batch whose requests are of very different lengths.
        attend_case("attend_batch", 64, 1, 8192, "ragged", 0, 32, 8, 128, "bf16", 16, "slot", 0.0),
        # Few requests with long contexts: the work lies along the cache.
        attend_case("attend_long", 2, 1, 131072, "even", 0, 64, 8, 128, "f16", 64, "head", 0.0),
        # Drafted tokens in 32 bits, each head with its own keys, a sliding window, some requests idle.
        attend_case("attend_drafts", 24, 3, 3000, "ragged", 1024, 12, 12, 80, "f32", 32, "head", 0.1),
    ]


def product_case(name, op, tokens, choices, experts, inner, outer, dtype, transposed, align):
    return {"name": name, "op": op, "tokens": tokens, "choices": choices, "experts": experts, "inner": inner, "outer": outer, "dtype": dtype,
            "transposed": transposed, "align": align}


def attend_case(name, requests, drafts, context, lengths, window, heads, key_heads, width, dtype, page, layout, idle):
    return {"name": name, "op": "attend", "requests": requests, "drafts": drafts, "context": context, "lengths": lengths, "window": window,
            "heads": heads, "key_heads": key_heads, "width": width, "dtype": dtype, "page": page, "layout": layout, "idle": idle}


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    while True:
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if rng.random() < 0.55:
            experts = spread(4, 256)
            case = product_case("", rng.choice(["product", "product", "weights"]), spread(1, 16384), min(rng.randint(1, 8), experts), experts,
                                spread(64, 5120), spread(64, 5120), dtype, rng.random() < 0.5, rng.choice([1, 1, 16, 64]))
            if rng.random() < 0.7:  # most models' widths
                case["inner"], case["outer"] = ((case[n] + 63) // 64 * 64 for n in ("inner", "outer"))
            if case["op"] == "weights":
                case["transposed"] = False
        else:
            key_heads = rng.choice([1, 2, 4, 8, 12, 16])
            case = attend_case("", spread(1, 256), rng.choice([1, 1, 1, 2, 4]), spread(1, 131072), rng.choice(["ragged", "ragged", "even"]),
                               rng.choice([0, 0, 0, 512, 4096]), key_heads * rng.choice([1, 2, 4, 7, 8, 16]), key_heads,
                               rng.choice([64, 80, 96, 128, 192, 256]), dtype, rng.choice([1, 16, 32, 64, 128]), rng.choice(["slot", "head"]),
                               rng.choice([0.0, 0.0, 0.2]))
        case.pop("name")
        need = work(case)
        if case["op"] == "attend" and 2 * case["requests"] * case["context"] * case["key_heads"] * case["width"] * SIZES[dtype] > 2 * MAX_BYTES:
            continue  # (the cache itself)
        if need["bytes"] <= MAX_BYTES and need["flops"] <= MAX_FLOPS[dtype]:
            return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def row_bound(case):
    """Rows that hold the sorted order of any routing, which a program knows before it."""
    n = case["tokens"] * case["choices"]
    return n + min(case["experts"], n) * (case["align"] - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return prepare_attend(case, g) if case["op"] == "attend" else prepare_products(case, g)


def prepare_products(case, g):
    experts, inner, outer, align, dtype = case["experts"], case["inner"], case["outer"], case["align"], TYPES[case["dtype"]]
    # distinct experts per token, some a little more in demand than others
    demand = 0.5 * torch.randn(experts, generator=g, device="cuda")
    ids = torch.topk(torch.randn(case["tokens"], experts, generator=g, device="cuda") + demand, case["choices"], dim=1)[1]
    count = torch.bincount(ids.reshape(-1), minlength=experts)
    padded = (count + align - 1) // align * align
    offsets = torch.cat([padded.new_zeros(1), torch.cumsum(padded, 0)])
    rows = row_bound(case)
    at = torch.arange(rows, device="cuda")
    segment = torch.searchsorted(offsets[1:], at, right=True).clamp(max=experts - 1)
    held = (at - offsets[segment] < count[segment])[:, None]

    def rows_of(width):  # rows without a token hold zeros
        return torch.randn(rows, width, generator=g, device="cuda", dtype=dtype).masked_fill_(~held, 0)

    state = {"case": case, "rows": rows, "offsets": offsets.to(torch.int32), "ends": offsets.tolist(), "x": rows_of(inner)}
    if case["op"] == "product":
        shape = (experts, outer, inner) if case["transposed"] else (experts, inner, outer)
        state["w"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(1 / math.sqrt(inner))
        state["y"] = torch.zeros(rows, outer, dtype=dtype, device="cuda")
    else:
        state["dy"] = rows_of(outer)
        state["dw"] = torch.empty(experts, inner, outer, dtype=dtype, device="cuda")
    return state


def prepare_attend(case, g):
    requests, drafts, page, heads, width, dtype = case["requests"], case["drafts"], case["page"], case["heads"], case["width"], TYPES[case["dtype"]]
    most = max(case["context"], drafts)
    if case["lengths"] == "even":
        length = torch.full((requests,), most, device="cuda")
    else:
        length = torch.randint(1, most + 1, (requests,), generator=g, device="cuda").clamp(min=drafts)
    owned = (length + page - 1) // page
    total = int(owned.sum())
    pages = total + total // 8 + 1  # some pages belong to nobody
    tables = torch.full((requests, (most + page - 1) // page), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(tables.shape[1], device="cuda")[None] < owned[:, None]
    tables[mine] = torch.randperm(pages, generator=g, device="cuda")[:total].to(torch.int32)
    # the queries of a request follow each other, the last one is its newest token's
    owners = torch.arange(requests, device="cuda").repeat_interleave(drafts)
    positions = length[owners] - drafts + torch.arange(requests * drafts, device="cuda") % drafts
    if case["idle"]:
        idle = torch.rand(requests, generator=g, device="cuda") < case["idle"]
        positions = torch.where(idle[owners], -1, positions)
    shape = (pages, page, case["key_heads"], width) if case["layout"] == "slot" else (pages, case["key_heads"], page, width)
    queries = requests * drafts
    # queries lie beside keys and values in the projection's output
    qkv = torch.randn(queries, heads + 2 * case["key_heads"], width, generator=g, device="cuda", dtype=dtype)
    state = {"case": case, "pages": pages, "tables": tables, "owners": owners.to(torch.int32), "positions": positions.to(torch.int32),
             "q": qkv[:, :heads].mul_(2), "k_cache": torch.randn(shape, generator=g, device="cuda", dtype=dtype),
             "v_cache": torch.randn(shape, generator=g, device="cuda", dtype=dtype),
             "out": torch.empty(queries, heads, width, dtype=dtype, device="cuda"), "logs": torch.empty(queries, heads, device="cuda")}
    if own:
        import cutt_amd as cutt
        space = cutt.cuttAttendPagesWorkspace(queries, heads, case["key_heads"], width, page, tables.shape[1], case["window"])
        state["workspace"] = torch.empty(space, dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"product": own_product, "weights": own_weights, "attend": own_attend}[op](state)
    return {"product": plain_product, "weights": plain_weights, "attend": plain_attend}[op](state)


def plain_product(state):
    x, w, y, ends = state["x"], state["w"], state["y"], state["ends"]
    for e in range(w.shape[0]):
        if ends[e] < ends[e + 1]:
            m = w[e].float()
            y[ends[e]:ends[e + 1]] = x[ends[e]:ends[e + 1]].float() @ (m.t() if state["case"]["transposed"] else m)
    return y


def plain_weights(state):
    x, dy, dw, ends = state["x"], state["dy"], state["dw"], state["ends"]
    for e in range(dw.shape[0]):
        dw[e] = x[ends[e]:ends[e + 1]].float().t() @ dy[ends[e]:ends[e + 1]].float()
    return dw


def plain_attend(state):
    case, q = state["case"], state["q"]
    queries, heads, width = q.shape
    key_heads, window = case["key_heads"], case["window"]
    positions, table = state["positions"].long(), state["tables"][state["owners"].long()].long()

    def cached(cache):  # [queries, key heads, tokens, width]
        c = cache[table.clamp(min=0)].float()
        c = c.permute(0, 3, 1, 2, 4) if case["layout"] == "slot" else c.permute(0, 2, 1, 3, 4)
        return c.reshape(queries, key_heads, -1, width)

    k = cached(state["k_cache"])
    at = torch.arange(k.shape[2], device=q.device)
    seen = at[None] <= positions[:, None]
    if window:
        seen &= at[None] > positions[:, None] - window
    scores = torch.matmul(q.float().reshape(queries, key_heads, -1, width), k.transpose(2, 3)) / math.sqrt(width)
    del k
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    logs = torch.logsumexp(scores, dim=3)
    p = torch.exp(scores - logs[..., None]).masked_fill_(~seen[:, None, None], 0)
    out = torch.matmul(p, cached(state["v_cache"]))
    return {"out": out.reshape(queries, heads, width).to(q.dtype), "logs": logs.reshape(queries, heads)}


# ---------------------------------------------------------------------------
# the same through this library
# ---------------------------------------------------------------------------
def checked(code, what):
    if code:
        import cutt_amd as cutt
        raise cutt.CuttError(code, what)


def stream():
    return torch.cuda.current_stream().cuda_stream


def row_type(case):
    import cutt_amd as cutt
    return {"f32": cutt.CUTT_F32, "f16": cutt.CUTT_F16, "bf16": cutt.CUTT_BF16}[case["dtype"]]


def own_product(state):
    import cutt_amd as cutt
    case, x, w, y = state["case"], state["x"], state["w"], state["y"]
    checked(cutt.cuttGroupedProduct(state["rows"], case["experts"], case["inner"], case["outer"], row_type(case), case["transposed"], stream(),
                                    state["offsets"].data_ptr(), x.data_ptr(), x.stride(0), w.data_ptr(), w.stride()[:2], y.data_ptr(), y.stride(0)),
            "cuttGroupedProduct")
    return y


def own_weights(state):
    import cutt_amd as cutt
    case, x, dy, dw = state["case"], state["x"], state["dy"], state["dw"]
    checked(cutt.cuttGroupedProductWeights(state["rows"], case["experts"], case["inner"], case["outer"], row_type(case), stream(),
                                           state["offsets"].data_ptr(), x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), dw.data_ptr(), dw.stride()[:2]),
            "cuttGroupedProductWeights")
    return dw


def own_attend(state):
    import cutt_amd as cutt
    case, q, k, out = state["case"], state["q"], state["k_cache"], state["out"]
    # strides in elements: of a page, a slot in it and a head
    cache = (k.stride(0), k.stride(1), k.stride(2)) if case["layout"] == "slot" else (k.stride(0), k.stride(2), k.stride(1))
    tables, space = state["tables"], state["workspace"]
    checked(cutt.cuttAttendPages(q.shape[0], tables.shape[0], case["heads"], case["key_heads"], case["width"], row_type(case), state["pages"], case["page"],
                                 tables.shape[1], case["window"], 1 / math.sqrt(case["width"]), stream(), tables.data_ptr(), state["owners"].data_ptr(),
                                 state["positions"].data_ptr(), q.data_ptr(), q.stride()[:2], k.data_ptr(), state["v_cache"].data_ptr(), cache,
                                 out.data_ptr(), out.stride()[:2], state["logs"].data_ptr(), space.data_ptr(), space.numel()), "cuttAttendPages")
    return {"out": out, "logs": state["logs"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and what it has to give
# ---------------------------------------------------------------------------
def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "attend":
        most = max(case["context"], case["drafts"])
        reach = min(case["window"] or most, most)
        if case["lengths"] == "even":
            seen = reach
        else:  # the mean over lengths of 1 to `most`
            seen = (reach * (reach + 1) / 2 + (most - reach) * reach) / most
        active = case["requests"] * (1 - case["idle"])
        rows = 2 * seen * case["key_heads"] * case["width"] * size + 4 * seen / case["page"]  # (a request's queries see the same rows)
        queries = case["requests"] * case["drafts"]
        return {"bytes": int(active * rows + queries * (case["heads"] * (2 * case["width"] * size + 4) + 8)),
                "flops": int(4 * active * case["drafts"] * seen * case["heads"] * case["width"])}
    n, experts = case["tokens"] * case["choices"], case["experts"]
    one = case["inner"] * case["outer"] * size
    rows = n * (case["inner"] + case["outer"]) * size + 4 * (experts + 1)
    hit = experts * (1 - (1 - case["choices"] / experts) ** case["tokens"])  # experts with a row, in the mean
    return {"bytes": int(rows + (hit if case["op"] == "product" else experts) * one), "flops": 2 * n * case["inner"] * case["outer"]}


def exact(case, seed):
    """From the definitions in 64 bits, segment by segment and request by request."""
    state = prepare(case, seed)
    if case["op"] == "attend":
        return exact_attend(case, state)
    ends = state["offsets"].tolist()
    x = state["x"]
    if case["op"] == "product":
        y = torch.zeros(state["y"].shape, dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            w = state["w"][e].double()
            torch.matmul(x[ends[e]:ends[e + 1]].double(), w.t() if case["transposed"] else w, out=y[ends[e]:ends[e + 1]])
        return y
    dw = torch.zeros(state["dw"].shape, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        for lo in range(ends[e], ends[e + 1], 4096):
            hi = min(lo + 4096, ends[e + 1])
            dw[e] += x[lo:hi].double().t() @ state["dy"][lo:hi].double()
    return dw


def exact_attend(case, state):
    q, page, key_heads = state["q"].double(), case["page"], case["key_heads"]
    queries, heads, width = q.shape
    out = torch.zeros(queries, heads, width, dtype=torch.float64, device="cuda")
    logs = torch.full((queries, heads), -math.inf, dtype=torch.float64, device="cuda")
    owners, positions = state["owners"].tolist(), state["positions"].tolist()
    for i in range(queries):
        p = positions[i]
        if p < 0:
            continue
        at = torch.arange(max(0, p - case["window"] + 1) if case["window"] else 0, p + 1, device="cuda")
        pages, slots = state["tables"][owners[i]][at // page].long(), at % page
        if case["layout"] == "slot":
            k, v = (state[n][pages, slots].double().transpose(0, 1).contiguous() for n in ("k_cache", "v_cache"))
        else:
            k, v = (state[n][pages, :, slots].double().transpose(0, 1).contiguous() for n in ("k_cache", "v_cache"))
        score = (q[i].reshape(key_heads, -1, 1, width) * k[:, None]).sum(3) if at.numel() < 64 else q[i].reshape(key_heads, -1, width) @ k.transpose(1, 2)
        score = score / width ** 0.5
        top = score.amax(2, keepdim=True)
        weight = torch.exp(score - top)
        total = weight.sum(2, keepdim=True)
        out[i] = ((weight / total) @ v).reshape(heads, width)
        logs[i] = (top + torch.log(total)).reshape(heads)
    return {"out": out, "logs": logs}
