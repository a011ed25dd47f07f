"""A small decoder layer with paged keys and values and routed experts, on the row operators of cutt_rows.h and the products of cutt_products.h.

    python examples/decoder_layer.py

Serving: prompts of several requests, then one token each, step by step.  cuttPageTables takes pages for the new tokens and names their
slots, and cuttPageStore puts their keys and values there.  For a prompt cuttPageLoad brings a request's keys and values back head by head and a transpose
plan turns the keys for the scores; a step's single tokens look at the pages where they are (cuttAttendPages).  The tokens go to their experts and
back (cuttExpertSort, cuttExpertDispatch, cuttExpertCombine), and there through the experts' weights (cuttGroupedProduct), no segment's end leaving the device.
Training: the same experts with the operators' gradients (cuttGroupedProductWeights among them) as autograd functions.  Both are compared with the same layer in
plain torch operations.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import cutt_amd as cutt  # noqa: E402


def check(code, what):
    if code != cutt.CUTT_SUCCESS:
        raise cutt.CuttError(code, what)


def stream():
    return torch.cuda.current_stream().cuda_stream


def row_type(t):
    return {torch.float32: cutt.CUTT_F32, torch.float16: cutt.CUTT_F16, torch.bfloat16: cutt.CUTT_BF16}[t.dtype]


# ---- rows to experts and back -------------------------------------------------------
class Routing:
    """Where the choices of a batch go: ids [tokens, choices] -> rows sorted by expert, every expert's segment a multiple of `align` rows."""

    def __init__(self, ids, experts, align):
        self.tokens, self.choices = ids.shape
        self.rows = cutt.cuttExpertRows(self.tokens, self.choices, experts, align)
        space = cutt.cuttExpertSortWorkspace(self.tokens, self.choices, experts)

        def ints(*shape):
            return torch.empty(*shape, dtype=torch.int32, device=ids.device)

        self.counts, self.offsets = ints(experts), ints(experts + 1)
        self.position, self.source = ints(self.tokens, self.choices), ints(self.rows)
        workspace = torch.empty(space, dtype=torch.uint8, device=ids.device)
        check(cutt.cuttExpertSort(self.tokens, self.choices, 0, experts, align, self.rows, ids.element_size(), stream(), ids.data_ptr(),
                                  self.counts.data_ptr(), self.offsets.data_ptr(), self.position.data_ptr(), self.source.data_ptr(),
                                  workspace.data_ptr(), space), "cuttExpertSort")


# Rows move and add up linearly, so the gradients' own gradients are the same operators again.
class Dispatch(torch.autograd.Function):
    """x [tokens, width] -> rows [routing.rows, width]"""

    @staticmethod
    def forward(ctx, x, routing):
        r, x = routing, x.contiguous()
        ctx.routing = r
        rows = torch.empty(r.rows, x.shape[1], dtype=x.dtype, device=x.device)
        check(cutt.cuttExpertDispatch(r.tokens, r.choices, r.rows, x.shape[1], x.element_size(), stream(), r.position.data_ptr(),
                                      r.source.data_ptr(), x.data_ptr(), x.stride(0), rows.data_ptr(), rows.stride(0)), "cuttExpertDispatch")
        return rows

    @staticmethod
    def backward(ctx, drows):
        return Gather.apply(drows, ctx.routing), None


class Gather(torch.autograd.Function):
    """rows [routing.rows, width] -> [tokens, width], the sums of the tokens' rows: the gradient of Dispatch, and Dispatch is its own."""

    @staticmethod
    def forward(ctx, rows, routing):
        r, rows = routing, rows.contiguous()
        ctx.routing = r
        out = torch.empty(r.tokens, rows.shape[1], dtype=rows.dtype, device=rows.device)
        check(cutt.cuttExpertDispatchBackward(r.tokens, r.choices, r.rows, rows.shape[1], row_type(rows), stream(), r.position.data_ptr(),
                                              rows.data_ptr(), rows.stride(0), out.data_ptr(), out.stride(0)), "cuttExpertDispatchBackward")
        return out

    @staticmethod
    def backward(ctx, dout):
        return Dispatch.apply(dout, ctx.routing), None


class Combine(torch.autograd.Function):
    """rows [routing.rows, width], weights [tokens, choices] in 32 bits -> [tokens, width]"""

    @staticmethod
    def forward(ctx, rows, weights, routing):
        ctx.routing = r = routing
        ctx.save_for_backward(rows, weights)
        rows, weights = rows.contiguous(), weights.contiguous()
        out = torch.empty(r.tokens, rows.shape[1], dtype=rows.dtype, device=rows.device)
        check(cutt.cuttExpertCombine(r.tokens, r.choices, r.rows, rows.shape[1], row_type(rows), stream(), r.position.data_ptr(),
                                     weights.data_ptr(), rows.data_ptr(), rows.stride(0), out.data_ptr(), out.stride(0)), "cuttExpertCombine")
        return out

    @staticmethod
    def backward(ctx, dout):
        rows, weights = ctx.saved_tensors
        return (*CombineGradients.apply(rows, weights, dout, ctx.routing, *ctx.needs_input_grad[:2]), None)


class CombineGradients(torch.autograd.Function):
    """The gradients of Combine for its rows and its weights, either of them None if it is not wanted."""

    @staticmethod
    def forward(ctx, rows, weights, dout, routing, of_rows, of_weights):
        ctx.routing = r = routing
        ctx.save_for_backward(rows, weights, dout)
        rows, weights, dout = rows.contiguous(), weights.contiguous(), dout.contiguous()
        drows = torch.empty_like(rows) if of_rows else None
        dweights = torch.empty_like(weights) if of_weights else None
        check(cutt.cuttExpertCombineBackward(r.tokens, r.choices, r.rows, rows.shape[1], row_type(rows), stream(), r.position.data_ptr(),
                                             r.source.data_ptr(), weights.data_ptr(), rows.data_ptr(), rows.stride(0), dout.data_ptr(), dout.stride(0),
                                             drows.data_ptr() if of_rows else 0, rows.stride(0), dweights.data_ptr() if of_weights else 0),
              "cuttExpertCombineBackward")
        return drows, dweights

    @staticmethod
    def backward(ctx, a, b):
        rows, weights, dout = ctx.saved_tensors
        r, drows, dweights, ddout = ctx.routing, None, None, []
        if a is not None:
            dweights = CombineGradients.apply(a, weights, dout, r, False, True)[1]
            ddout.append(Combine.apply(a, weights, r))
        if b is not None:
            drows = CombineGradients.apply(rows, b, dout, r, True, False)[0]
            ddout.append(Combine.apply(rows, b, r))
        return drows, dweights, sum(ddout[1:], ddout[0]), None, None, None


class Product(torch.autograd.Function):
    """rows [routing.rows, inner], every segment's times its expert's weights: [experts, inner, outer], or transposed [experts, outer, inner].  What is behind
    the last segment is not written: no row comes from there."""

    @staticmethod
    def forward(ctx, rows, weights, routing, transposed):
        rows, weights = rows.contiguous(), weights.contiguous()
        ctx.routing, ctx.transposed = routing, transposed
        ctx.save_for_backward(rows, weights)
        experts, outer = weights.shape[0], weights.shape[1 if transposed else 2]
        out = torch.empty(routing.rows, outer, dtype=rows.dtype, device=rows.device)
        check(cutt.cuttGroupedProduct(routing.rows, experts, rows.shape[1], outer, row_type(rows), transposed, stream(), routing.offsets.data_ptr(),
                                      rows.data_ptr(), rows.stride(0), weights.data_ptr(), weights.stride()[:2], out.data_ptr(), out.stride(0)),
              "cuttGroupedProduct")
        return out

    @staticmethod
    def backward(ctx, dout):
        rows, weights = ctx.saved_tensors
        drows = Product.apply(dout, weights, ctx.routing, not ctx.transposed) if ctx.needs_input_grad[0] else None
        sides = (dout, rows) if ctx.transposed else (rows, dout)
        return drows, WeightsGradient.apply(*sides, ctx.routing) if ctx.needs_input_grad[1] else None, None, None


class WeightsGradient(torch.autograd.Function):
    """rows [routing.rows, inner], dout [routing.rows, outer] -> [experts, inner, outer], the sums of a segment's outer products: Product's gradient for its
    weights, and Product gives its own."""

    @staticmethod
    def forward(ctx, rows, dout, routing):
        rows, dout = rows.contiguous(), dout.contiguous()
        ctx.routing = routing
        ctx.save_for_backward(rows, dout)
        dw = torch.empty(routing.counts.numel(), rows.shape[1], dout.shape[1], dtype=rows.dtype, device=rows.device)
        check(cutt.cuttGroupedProductWeights(routing.rows, dw.shape[0], dw.shape[1], dw.shape[2], row_type(rows), stream(), routing.offsets.data_ptr(),
                                             rows.data_ptr(), rows.stride(0), dout.data_ptr(), dout.stride(0), dw.data_ptr(), dw.stride()[:2]),
              "cuttGroupedProductWeights")
        return dw

    @staticmethod
    def backward(ctx, g):
        rows, dout = ctx.saved_tensors
        return Product.apply(dout, g, ctx.routing, True), Product.apply(rows, g, ctx.routing, False), None


class Experts:
    """A router and its experts, each two products with a nonlinearity between."""

    def __init__(self, width, hidden, experts, choices, align=16, dtype=torch.float32):
        def weight(*shape):
            return (torch.randn(*shape, device="cuda") / math.sqrt(shape[-2])).to(dtype).requires_grad_()

        self.router, self.up, self.down = weight(width, experts), weight(experts, width, hidden), weight(experts, hidden, width)
        self.experts, self.choices, self.align = experts, choices, align

    def parameters(self):
        return [self.router, self.up, self.down]

    def route(self, x):
        top, ids = torch.topk((x @ self.router).float(), self.choices, dim=1)
        return ids, torch.softmax(top, dim=1)

    def __call__(self, x):
        ids, weights = self.route(x)
        routing = Routing(ids, self.experts, self.align)
        inside = torch.nn.functional.gelu(Product.apply(Dispatch.apply(x, routing), self.up, routing, False))
        return Combine.apply(Product.apply(inside, self.down, routing, False), weights, routing)

    def plain(self, x):
        ids, weights = self.route(x)
        out = torch.zeros_like(x)
        for e in range(self.experts):
            token, k = torch.where(ids == e)
            y = torch.nn.functional.gelu(x[token] @ self.up[e]) @ self.down[e]
            out = out.index_add(0, token, y * weights[token, k][:, None].to(y.dtype))
        return out


# ---- keys and values in pages ----------------------------------------------------------
class PagedCache:
    """Keys and values of `requests` requests in pages [pages, heads, page, width], in 32 bits."""

    def __init__(self, requests, heads, width, page, pages, most):
        self.heads, self.width, self.page, self.pages = heads, width, page, pages
        self.k = torch.zeros(pages, heads, page, width, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.tables = torch.full((requests, (most + page - 1) // page), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, device="cuda").to(torch.int32)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
        # elements from page to page, slot to slot, head to head
        self.strides = (self.k.stride(0), self.k.stride(2), self.k.stride(1))

    def extend(self, added, tokens):
        """Pages and slots for `added` new tokens per request, `tokens` in all: (slots, positions)."""
        requests = added.numel()
        starts = torch.empty(requests + 1, dtype=torch.int32, device="cuda")
        used = torch.empty(1, dtype=torch.int32, device="cuda")
        slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        positions = torch.empty(tokens, dtype=torch.int32, device="cuda")
        check(cutt.cuttPageTables(requests, self.page, self.tables.shape[1], self.free.numel(), tokens, stream(), self.lengths.data_ptr(), added.data_ptr(),
                                  self.free.data_ptr(), self.tables.data_ptr(), starts.data_ptr(), used.data_ptr(), slots.data_ptr(),
                                  positions.data_ptr()), "cuttPageTables")
        taken = int(used)
        if taken > self.free.numel():
            raise RuntimeError("out of pages")
        self.free = self.free[taken:].contiguous()
        self.lengths = self.lengths + added
        return slots, positions

    def store(self, slots, k, v):
        """k, v [tokens, heads, width], any strides of the first two (both the same)."""
        check(cutt.cuttPageStore(slots.numel(), self.heads, self.width, 4, self.pages, self.page, stream(), slots.data_ptr(), k.data_ptr(), v.data_ptr(),
                                 k.stride()[:2], self.k.data_ptr(), self.v.data_ptr(), self.strides), "cuttPageStore")

    def load(self, request, length):
        """Keys and values of a request's tokens, [heads, length, width]."""
        at = torch.arange(length, device="cuda")
        slots = self.tables[request, at // self.page].long() * self.page + at % self.page
        k = torch.empty(self.heads, length, self.width, device="cuda")
        v = torch.empty_like(k)
        check(cutt.cuttPageLoad(length, self.heads, self.width, 4, self.pages, self.page, stream(), slots.data_ptr(), k.data_ptr(), v.data_ptr(),
                                (k.stride(1), k.stride(0)), self.k.data_ptr(), self.v.data_ptr(), self.strides), "cuttPageLoad")
        return k, v


    def attend(self, q, owners, positions):
        """q [tokens, heads, width] of requests `owners` at `positions`, over the pages: [tokens, heads, width]."""
        tokens, heads, width = q.shape
        out = torch.empty(tokens, heads, width, device="cuda")
        space = cutt.cuttAttendPagesWorkspace(tokens, heads, self.heads, width, self.page, self.tables.shape[1], 0)
        workspace = torch.empty(space, dtype=torch.uint8, device="cuda")
        check(cutt.cuttAttendPages(tokens, self.tables.shape[0], heads, self.heads, width, cutt.CUTT_F32, self.pages, self.page, self.tables.shape[1], 0,
                                   1 / math.sqrt(width), stream(), self.tables.data_ptr(), owners.data_ptr(), positions.data_ptr(), q.data_ptr(),
                                   q.stride()[:2], self.k.data_ptr(), self.v.data_ptr(), self.strides, out.data_ptr(), out.stride()[:2], 0,
                                   workspace.data_ptr(), space), "cuttAttendPages")
        return out


def turned(k):
    """[heads, length, width] -> [heads, width, length], by a transpose of the library."""
    heads, length, width = k.shape
    if min(heads, length, width) < 2:  # (its extents are 2 and more)
        return k.transpose(1, 2).contiguous()
    out = torch.empty(heads, width, length, device="cuda")
    check(cutt.cuttExecuteNoAlloc(3, (width, length, heads), (1, 0, 2), 4, stream(), k.data_ptr(), out.data_ptr()), "cuttExecuteNoAlloc")
    return out


class DecoderLayer:
    def __init__(self, width, heads, experts, choices):
        self.heads, self.size = heads, width // heads
        self.qkv = torch.randn(width, 3 * width, device="cuda") / math.sqrt(width)
        self.out = torch.randn(width, width, device="cuda") / math.sqrt(width)
        self.experts = Experts(width, 2 * width, experts, choices)

    def project(self, x):
        qkv = (x @ self.qkv).view(x.shape[0], 3 * self.heads, self.size)
        return qkv[:, :self.heads], qkv[:, self.heads:2 * self.heads], qkv[:, 2 * self.heads:]

    def attend(self, q, kt, v, before):
        """q [tokens, heads, size] at positions before, before + 1, ...; kt [heads, size, length], v [heads, length, size]"""
        scores = torch.matmul(q.transpose(0, 1).contiguous(), kt) / math.sqrt(self.size)
        here = before + torch.arange(q.shape[0], device="cuda")[:, None]
        scores = scores.masked_fill(torch.arange(v.shape[1], device="cuda")[None] > here, float("-inf"))
        return torch.matmul(torch.softmax(scores, dim=-1), v).transpose(0, 1).reshape(q.shape[0], -1) @ self.out

    @torch.no_grad()
    def step(self, x, cache, added):
        """x [tokens, width]: the new tokens of all requests, `added` of each (a list)."""
        before = cache.lengths.tolist()
        slots, positions = cache.extend(torch.tensor(added, dtype=torch.int32, device="cuda"), x.shape[0])
        q, k, v = self.project(x)
        cache.store(slots, k, v)
        if max(added) == 1:
            owners = torch.tensor([b for b, n in enumerate(added) if n], dtype=torch.int32, device="cuda")
            x = x + cache.attend(q, owners, positions).reshape(x.shape[0], -1) @ self.out
            return x + self.experts(x)
        parts, at = [], 0
        for b, n in enumerate(added):
            if n:
                ks, vs = cache.load(b, before[b] + n)
                parts.append(self.attend(q[at:at + n], turned(ks), vs, before[b]))
                at += n
        x = x + torch.cat(parts)
        return x + self.experts(x)

    @torch.no_grad()
    def plain(self, x):
        """All tokens of one request at once."""
        q, k, v = self.project(x)
        kt = k.permute(1, 2, 0).contiguous()
        x = x + self.attend(q, kt, v.transpose(0, 1).contiguous(), 0)
        return x + self.experts.plain(x)


def serve(width=256, heads=4, experts=8, choices=2, prompts=(37, 1, 64, 0, 5), steps=6, page=16, seed=0):
    """The largest difference between requests served step by step and the same tokens in one plain pass, and the largest output."""
    torch.manual_seed(seed)
    layer = DecoderLayer(width, heads, experts, choices)
    most = max(prompts) + steps
    cache = PagedCache(len(prompts), heads, width // heads, page, len(prompts) * ((most + page - 1) // page), most)
    tokens = [torch.randn(n + steps, width, device="cuda") for n in prompts]
    got = [[] for _ in prompts]
    at = [0] * len(prompts)
    for step in range(steps + 1):
        added = list(prompts) if step == 0 else [1] * len(prompts)
        y = layer.step(torch.cat([t[p:p + n] for t, p, n in zip(tokens, at, added)]), cache, added)
        for b, part in enumerate(y.split(added)):
            got[b].append(part)
            at[b] += added[b]
    worst = biggest = 0.0
    for t, g in zip(tokens, got):
        want = layer.plain(t)
        worst = max(worst, float((torch.cat(g) - want).abs().max()))
        biggest = max(biggest, float(want.abs().max()))
    return worst, biggest


def train(width=128, hidden=256, experts=8, choices=3, tokens=100, dtype=torch.float32, seed=0, second=False):
    """The largest relative difference (norms) between the gradients through the operators and through plain torch operations.  second: between the
    gradients of the gradients' products with a fixed direction."""
    torch.manual_seed(seed)
    layer = Experts(width, hidden, experts, choices, dtype=dtype)
    x = torch.randn(tokens, width, device="cuda").to(dtype).requires_grad_()
    goal = torch.randn(tokens, width, device="cuda")
    leaves = [x] + layer.parameters()
    along = [torch.randn_like(t) for t in leaves]
    grads = []
    for way in (layer, layer.plain):
        loss = ((way(x).float() - goal) ** 2).mean()
        grad = torch.autograd.grad(loss, leaves, create_graph=second)
        if second:
            grad = torch.autograd.grad(sum((g * d).sum() for g, d in zip(grad, along)), leaves)
        grads.append(grad)
    return max(float((a.double() - b.double()).norm() / b.double().norm()) for a, b in zip(*grads))


if __name__ == "__main__":
    worst, biggest = serve()
    print("serving: largest difference to one plain pass %.2g, largest output %.2g" % (worst, biggest))
    print("training: gradients differ from plain ones by %.2g (float), %.2g (bfloat16)" % (train(), train(dtype=torch.bfloat16)))
