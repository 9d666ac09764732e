"""Many sequences in one paged cache of 8 or 4 bits: the operators of a serving step between the packed linears.

  plan_step     page tables, positions and slots of a step, built on the GPU from the requests' lengths
  rope_append   rotary embedding, and the step's keys and values into the cache (e4m3, one power-of-two scale per page and head; or
                e2m1, one bf16 scale per token and head, with a Hadamard transform of queries and keys)
  attention     grouped-query causal attention over the cache, from single tokens to prompts
  unpack        pages of the 4-bit cache as keys and values
  PagedCache    the buffers that a server keeps: caches of all layers, page tables, free pages

Requests are rows: a step gives each of them as many tokens as it likes (none, one, a prompt), and the step's tokens stand one request
after the other.  Nothing touches the host, so that a step can be captured in a CUDA graph.  Lengths, tables and slots are int32.
No operator here has a gradient: results of inputs that require one do not.
"""
import typing

import torch

from . import _lib, ops

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_host = _lib.host
_HALF = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


class LayerCache(typing.NamedTuple):
    """One layer's cache: k, v float8_e4m3fn [pages, kv_heads, page_size, head_dim]; k_scale, v_scale float32 [pages, kv_heads], powers of
    two.  The value of an element is element * scale."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class LayerCache4(typing.NamedTuple):
    """One layer's cache in 4 bits: k, v uint8 [pages, kv_heads, page_size, head_dim / 2], two e2m1 codes in a byte, the even dimension in its low half;
    k_scale, v_scale bfloat16 [pages, kv_heads, page_size], between 2^-100 and 2^119 (NaN: so are the token's values).  The value of an element is
    its code's (0, 0.5, 1, 1.5, 2, 3, 4, 6, and negative with the highest bit) * scale.  A key is held as H k / 8, H the Hadamard matrix of head_dim rows in
    Sylvester's order; a query that meets it has to be H q * 8 / head_dim, as `rope_append` returns it."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class StepPlan(typing.NamedTuple):
    """What a step's operators need: starts [requests + 1], positions and slots [max_tokens], seen, lengths [requests], count [1]."""
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    seen: torch.Tensor
    lengths: torch.Tensor
    count: torch.Tensor


def _int32(what, name, t, dev, *shape):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != dev or tuple(t.shape) != shape or not t.is_contiguous():
        raise _lib.HTRError(f"{what}: {name} must be a contiguous int32 tensor {list(shape)} on {dev}")


def _tables(what, tables, dev, requests):
    if tables.dtype != torch.int32 or tables.device != dev or tables.dim() != 2 or tables.shape[0] != requests or tables.shape[1] < 1 or \
            tables.stride(1) != 1 or (requests > 1 and tables.stride(0) < tables.shape[1]):
        raise _lib.HTRError(f"{what}: tables must be int32 [{requests}, pages of a request] on {dev} with rows that do not overlap")
    return max(tables.stride(0), tables.shape[1])


def _status(what, status, dev):
    if status is None:
        return None
    _int32(what, "status", status, dev, 1)
    return status.data_ptr()


def _cache(what, cache, dev):
    """Pages, heads, page size, head dimensions of a layer's cache, and whether it is in 4 bits."""
    if cache[0].dtype == torch.uint8:
        return *_cache4(what, cache, dev), True
    return *_cache8(what, cache, dev), False


def _cache4(what, cache, dev):
    k, v, ks, vs = cache
    if k.dtype != torch.uint8 or k.dim() != 4 or k.device != dev or not k.is_contiguous() or v.dtype != k.dtype or v.shape != k.shape or \
            v.device != dev or not v.is_contiguous():
        raise _lib.HTRError(f"{what}: k and v must be contiguous uint8 [pages, kv_heads, page_size, head_dim / 2] on {dev}")
    pages, heads, page, dim = *k.shape[:3], 2 * k.shape[3]
    if pages < 1 or heads < 1 or page not in PAGE_SIZES or dim not in HEAD_DIMS:
        raise _lib.HTRError(f"{what}: pages of {PAGE_SIZES} tokens and heads of {HEAD_DIMS} are supported, got {page} and {dim}")
    for s in (ks, vs):
        if s.dtype != torch.bfloat16 or s.device != dev or tuple(s.shape) != (pages, heads, page) or not s.is_contiguous():
            raise _lib.HTRError(f"{what}: scales must be contiguous bfloat16 [{pages}, {heads}, {page}] on {dev}")
    return pages, heads, page, dim


def _cache8(what, cache, dev):
    k, v, ks, vs = cache
    if k.dtype != torch.float8_e4m3fn or k.dim() != 4 or k.device != dev or not k.is_contiguous() or v.dtype != k.dtype or v.shape != k.shape or \
            v.device != dev or not v.is_contiguous():
        raise _lib.HTRError(f"{what}: k and v must be contiguous float8_e4m3fn [pages, kv_heads, page_size, head_dim] on {dev}")
    pages, heads, page, dim = k.shape
    if pages < 1 or heads < 1 or page not in PAGE_SIZES or dim not in HEAD_DIMS:
        raise _lib.HTRError(f"{what}: pages of {PAGE_SIZES} tokens and heads of {HEAD_DIMS} are supported, got {page} and {dim}")
    for s in (ks, vs):
        if s.dtype != torch.float32 or s.device != dev or tuple(s.shape) != (pages, heads) or not s.is_contiguous():
            raise _lib.HTRError(f"{what}: scales must be contiguous float32 [{pages}, {heads}] on {dev}")
    return pages, heads, page, dim


def plan_step(lengths, new, tables, free, count, page_size, max_tokens, lengths_out=None, count_out=None, status=None):
    """The tables and slots of one step.

    lengths [requests]: tokens that each request has in the cache; new [requests]: tokens that it adds (0: none; negative: it is over and its
    pages come back); tables [requests, pages of a request]; free [pages], of which the first count[0] are free.  A request that grows gets
    the pages it lacks, in the order of the requests: first those that came back in this step, then from the top of `free`.  `tables` and `free`
    are updated in place.  A page stands in one table and at one place of it: the pages of a request that is over come back whoever else has them.
    Returns a StepPlan: starts (the first token of each request in the step), positions and slots of max_tokens tokens
    (-1: not served, and behind the last), seen (tokens in the cache after the step of a request that adds some, else 0), and the lengths
    and count after the step, in new tensors or in lengths_out / count_out (which may be lengths and count themselves).

    A request that cannot be served keeps its length and its tokens get -1; status [1], if given, then gets a bit: 1 no pages left (this request
    and later ones that need pages), 2 its table is full, 4 its length is negative or beyond its table, 8 tokens beyond max_tokens."""
    what = "plan_step"
    plan = _host.plan_step(lengths, new, tables, free, count, page_size, max_tokens, lengths_out, count_out, status)    # the usual case; None: whatever it does not take
    if plan is not None:
        return StepPlan._make(plan)
    if not lengths.is_cuda:
        raise _lib.HTRError("plan_step has no CPU path: tensors must live on a CUDA device")
    dev, R, T = lengths.device, lengths.numel(), int(max_tokens)
    _int32(what, "lengths", lengths, dev, R)
    _int32(what, "new", new, dev, R)
    _int32(what, "count", count, dev, 1)
    _int32(what, "free", free, dev, free.numel())
    if page_size not in PAGE_SIZES:
        raise _lib.HTRError(f"plan_step: pages of {PAGE_SIZES} tokens are supported, got {page_size}")
    if R < 1 or free.numel() < 1 or T < 0:
        raise _lib.HTRError("plan_step: wants at least one request and one page, and max_tokens >= 0")
    stride = _tables(what, tables, dev, R)
    for name, t, n in (("lengths_out", lengths_out, R), ("count_out", count_out, 1)):
        if t is not None:
            _int32(what, name, t, dev, n)
    flat = torch.empty(2 * R + 1 + 2 * T, dtype=torch.int32, device=dev)
    starts, seen, positions, slots = flat[:R + 1], flat[R + 1:2 * R + 1], flat[2 * R + 1:2 * R + 1 + T], flat[2 * R + 1 + T:]
    lengths_out = torch.empty_like(lengths) if lengths_out is None else lengths_out
    count_out = torch.empty_like(count) if count_out is None else count_out
    with torch.cuda.device(dev):
        rc = _lib.lib.htr_page_plan(lengths.data_ptr(), new.data_ptr(), R, tables.data_ptr(), stride, tables.shape[1], free.data_ptr(), free.numel(),
                                    count.data_ptr(), page_size, T, starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), seen.data_ptr(),
                                    lengths_out.data_ptr(), count_out.data_ptr(), _status(what, status, dev), torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc, "htr_page_plan")
    return StepPlan(starts, positions, slots, seen, lengths_out, count_out)


def rope_append(qkv, positions, slots, cos, sin, cache, q_heads, status=None, layout="interleaved"):
    """Rotary embedding of a step's queries and keys, and its keys and values into one layer's cache (LayerCache or LayerCache4).

    qkv [tokens, (q_heads + 2 kv_heads) * head_dim] bf16 or fp16 (rows may be strided); positions, slots [tokens] as `plan_step` gives them; cos, sin
    float32 [rows, head_dim / 2], a row per position, for interleaved pairs.  Returns the rotated queries [tokens, q_heads, head_dim].

    A token with slot -1 is not written and its query is zero; so is one whose slot or position lies outside the buffers (status 16).
    The tokens of one page stand one after the other in rising slots, as `plan_step` lays them out, within page_size tokens of the step (tokens that are not
    written may lie between them).  In 8 bits, from a slot that does not rise on, that page's are not written; in 4, a token is not whose slot does not lie above
    those of its page among the page_size - 1 tokens before it (status 16 both).  A slot that comes again farther on is the caller's to avoid: what it then holds may be
    the codes of one token under the scale of the other.

    8 bits: a page's scale is the smallest power of two (at least 2^-100) under which all of its tokens lie within e4m3 (448); it begins anew with the
    page's first place, and where a later token makes it grow the older ones are rescaled.  Infinities are held as the largest value, NaN as NaN.

    4 bits: pairs may also be halves (layout "half": dimensions i and i + r / 2), and r, twice the columns of cos and sin, a part of the
    head that is a multiple of 16: the first r dimensions are rotated.  The queries come back as H q * 8 / head_dim for the keys of such a cache (see
    LayerCache4; sums are float32, and where tokens times heads reach 32768, of elements that are cut at 2^-20 of what they are: the code of an element beside a tie may depend
    on how many tokens the step has; fp16 ones whose sums leave its range become infinite, and rows of bf16 ones beyond 2^124 may become infinite or NaN).  A token's scale is bf16(largest / 6), its codes are the
    nearest, ties to the even code.  Infinities among values are held as the largest value, 6 * 2^119, as is all that lies beyond it; a row of a head that has a NaN is
    NaN as a whole, and so is one of queries or keys that has an infinity; finite keys stay so under cosines and sines of a magnitude up to 8."""
    what = "rope_append"
    q = _host.rope_append(qkv, positions, slots, cos, sin, cache, q_heads, status, layout)
    if q is not None:
        return q
    if not qkv.is_cuda:
        raise _lib.HTRError("rope_append has no CPU path: tensors must live on a CUDA device")
    dev = qkv.device
    pages, kv_heads, page, dim, four = _cache(what, cache, dev)
    q_heads = int(q_heads)
    if layout not in ("interleaved", "half") or (layout == "half" and not four):
        raise _lib.HTRError(f"rope_append: layout is \"interleaved\", or for a cache of 4 bits \"half\", got {layout!r}")
    if qkv.dtype not in _HALF or qkv.dim() != 2 or q_heads < 1 or qkv.shape[1] != (q_heads + 2 * kv_heads) * dim:
        raise _lib.HTRError(f"rope_append: qkv must be bf16 or fp16 [tokens, {(q_heads + 2 * kv_heads) * dim}]")
    T = qkv.shape[0]
    if qkv.stride(1) != 1 or (T > 1 and (qkv.stride(0) < qkv.shape[1] or qkv.stride(0) % 8)) or qkv.data_ptr() % 16:
        qkv = qkv.contiguous() if not qkv.is_contiguous() else qkv.clone()
    _int32(what, "positions", positions, dev, T)
    _int32(what, "slots", slots, dev, T)
    for t in (cos, sin):
        if t.dtype != torch.float32 or t.device != dev or t.dim() != 2 or t.shape != cos.shape or not t.is_contiguous() or \
                (t.shape[1] not in range(8, dim // 2 + 1, 8) if four else t.shape[1] != dim // 2):
            raise _lib.HTRError(f"rope_append: cos and sin must be contiguous float32 [positions, {'a multiple of 8 up to ' if four else ''}{dim // 2}] on {dev}")
    q = torch.empty((T, q_heads, dim), dtype=qkv.dtype, device=dev)
    if T == 0:
        return q
    with torch.cuda.device(dev):
        if four:
            rc = _lib.lib.htr_paged4_append(qkv.data_ptr(), _HALF[qkv.dtype], max(qkv.stride(0), qkv.shape[1]), positions.data_ptr(), slots.data_ptr(), T,
                                            cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1], int(layout == "half"), q_heads, kv_heads, dim,
                                            *[t.data_ptr() for t in cache], pages, page, q.data_ptr(), _status(what, status, dev),
                                            torch.cuda.current_stream(dev).cuda_stream)
            _lib.check(rc, "htr_paged4_append")
            return q
        rc = _lib.lib.htr_paged_append(qkv.data_ptr(), _HALF[qkv.dtype], max(qkv.stride(0), qkv.shape[1]), positions.data_ptr(), slots.data_ptr(), T,
                                       cos.data_ptr(), sin.data_ptr(), cos.shape[0], q_heads, kv_heads, dim, cache[0].data_ptr(), cache[1].data_ptr(),
                                       cache[2].data_ptr(), cache[3].data_ptr(), pages, page, q.data_ptr(), _status(what, status, dev),
                                       torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc, "htr_paged_append")
    return q


def attention(q, starts, seen, tables, cache, max_new, scale=None, out=None, status=None):
    """Causal grouped-query attention of a step's tokens over one layer's cache (LayerCache, or LayerCache4 with queries that `rope_append` made for it).

    q [tokens, q_heads, head_dim] bf16 or fp16; starts [requests + 1] and seen [requests] as `plan_step` gives them: of the n tokens
    [starts[r], starts[r + 1]) of request r the i-th stands at position seen[r] - n + i and sees the cached positions up to its own; one that
    sees nothing gets zeros.  max_new: at least the largest n (tokens of a request beyond it are not computed).  scale: of the scores, 1 / sqrt(head_dim) by default.
    Returns `out`, or a new tensor like q; its rows behind starts[-1] are left as they are.  A table entry that is no page hides its
    tokens (status 32).  Status 64: a wait inside the kernel ran out (about two seconds); the rows that it concerns are NaN.

    Sums are float32.  A probability times the scale of its values' page is rounded to fp16: by 2^-11 of itself down to 2^-26 of the row's largest
    (18 nats), below by up to 2^-37 of that.  For bf16 that is less than the rounding of the output, for fp16 as much.  Where a request adds many
    rows, elements of a query below 2^-9 (fp16: 2^-6) of its largest are held to 2^-17 of the largest.  Scales of the values of one request and head
    that lie 2^110 or more apart lose the probabilities under the smaller ones.

    Over a cache of 4 bits it is the scale of the value (where a request adds many rows, the largest of 16 neighbours, seen or not, as far as it lies less than 2^5
    above), and fp16 holds 2^-11 down to 2^-18 of the row's largest (12 nats), below by up to 2^-29 of that; queries are held to 28 binades, and keys and values exactly.
    Many rows take up to about twice as long over neighbours whose scales differ by more (keys: 2^13).

    Many rows a request are fast for up to 1024 requests and 256 query heads per key/value head; beyond, 16 rows at a time go over the cache.  Which kernel serves goes by max_new and
    the tables' width for all requests of a call: a piece of a prompt and many single tokens are faster in calls of their own."""
    what = "attention"
    y = _host.attention(q, starts, seen, tables, cache, max_new, scale, out, status)
    if y is not None:
        return y
    if not q.is_cuda:
        raise _lib.HTRError("attention has no CPU path: tensors must live on a CUDA device")
    dev, R = q.device, seen.numel()
    pages, kv_heads, page, dim, four = _cache(what, cache, dev)
    if q.dtype not in _HALF or q.dim() != 3 or q.shape[2] != dim or q.shape[1] < 1 or q.shape[1] % kv_heads:
        raise _lib.HTRError(f"attention: q must be bf16 or fp16 [tokens, a multiple of {kv_heads} heads, {dim}]")
    T, q_heads = q.shape[:2]
    if R < 1 or int(max_new) < 1:
        raise _lib.HTRError("attention: wants at least one request, and max_new >= 1")
    _int32(what, "starts", starts, dev, R + 1)
    _int32(what, "seen", seen, dev, R)
    stride = _tables(what, tables, dev, R)
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.contiguous() if not q.is_contiguous() else q.clone()
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype != q.dtype or out.shape != q.shape or out.device != dev or not out.is_contiguous():
        raise _lib.HTRError("attention: `out` must be a contiguous tensor like q")
    if T == 0:
        return out
    most = min(int(max_new), T)
    with torch.cuda.device(dev):
        need_of = _lib.lib.htr_paged4_attention_workspace_bytes if four else _lib.lib.htr_paged_attention_workspace_bytes
        need = need_of(T, R, q_heads, kv_heads, dim, most, tables.shape[1], page)      # (by the device's SMs)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        entry = _lib.lib.htr_paged4_attention if four else _lib.lib.htr_paged_attention
        rc = entry(q.data_ptr(), _HALF[q.dtype], T, starts.data_ptr(), seen.data_ptr(), R, tables.data_ptr(), stride, tables.shape[1], cache[0].data_ptr(),
                   cache[1].data_ptr(), cache[2].data_ptr(), cache[3].data_ptr(), pages, page, q_heads, kv_heads, dim, most,
                   float(dim ** -0.5 if scale is None else scale), out.data_ptr(), _status(what, status, dev), None if work is None else work.data_ptr(), need,
                   torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc, "htr_paged4_attention" if four else "htr_paged_attention")
    return out


def unpack(cache, pages, dtype=torch.bfloat16):
    """The keys and values that pages of a LayerCache4 stand for: (k, v) [len(pages), kv_heads, page_size, head_dim] in dtype (bf16, fp16 or float32), rounded
    once; keys are turned back (H k / 8 to k; float32 sums).  pages: int32; one that is none gives zeros."""
    both = _host.unpack(cache, pages, dtype)
    if both is not None:
        return both
    if not pages.is_cuda:
        raise _lib.HTRError("unpack has no CPU path: tensors must live on a CUDA device")
    dev = pages.device
    count, kv_heads, page, dim = _cache4("unpack", cache, dev)
    _int32("unpack", "pages", pages, dev, pages.numel())
    if dtype not in ops._DTYPES:
        raise _lib.HTRError("unpack: dtype must be bf16, fp16 or float32")
    out = [torch.empty((pages.numel(), kv_heads, page, dim), dtype=dtype, device=dev) for _ in range(2)]
    with torch.cuda.device(dev):
        rc = _lib.lib.htr_paged4_unpack(*[t.data_ptr() for t in cache], count, kv_heads, page, dim, pages.data_ptr(), pages.numel(), out[0].data_ptr(),
                                        out[1].data_ptr(), ops._DTYPES[dtype], torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc, "htr_paged4_unpack")
    return tuple(out)


class PagedCache:
    """What a server keeps from step to step: the caches of all layers, the requests' page tables and lengths, and the free pages."""

    def __init__(self, layers, kv_heads, head_dim, pages, page_size, requests, max_len, device, bits=8):
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise _lib.HTRError(f"PagedCache: pages of {PAGE_SIZES} tokens and heads of {HEAD_DIMS} are supported, got {page_size} and {head_dim}")
        if min(layers, kv_heads, pages, requests, max_len) < 1:
            raise _lib.HTRError("PagedCache: layers, kv_heads, pages, requests and max_len must be positive")
        if bits not in (4, 8):
            raise _lib.HTRError(f"PagedCache: 8 or 4 bits are supported, got {bits}")
        shape = (layers, pages, kv_heads, page_size, head_dim * bits // 8)
        self.page_size, self.device, self.bits = page_size, device, bits
        self.k, self.v = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        if bits == 8:
            self.k, self.v = self.k.view(torch.float8_e4m3fn), self.v.view(torch.float8_e4m3fn)
        scales = (shape[:3], torch.float32) if bits == 8 else (shape[:4], torch.bfloat16)
        self.k_scale, self.v_scale = (torch.ones(scales[0], dtype=scales[1], device=device) for _ in range(2))
        self.tables = torch.full((requests, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)       # page 0 is taken first
        self.count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.cos = self.sin = None                            # angles of the positions, where a model lays them out (PackedDecoder.paged_cache)

    def layer(self, i):
        return (LayerCache if self.bits == 8 else LayerCache4)(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])

    def plan(self, new, max_tokens):
        """`plan_step` on this cache's own buffers, which are updated in place: new [requests] int32, tokens that each adds (negative: it is over)."""
        return plan_step(self.lengths, new, self.tables, self.free, self.count, self.page_size, max_tokens, lengths_out=self.lengths, count_out=self.count,
                         status=self.status)
