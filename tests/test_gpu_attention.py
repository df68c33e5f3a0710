"""GPU: norm with rotation, paged cache and paged attention against plain statements of their definitions in 64 bits.

Tolerances, from the arithmetic (u = half a step of a type: bf16 2^-8, fp16 2^-11, fp32 2^-24):
  attention   A = sum_j softmax_j |v_j|.  The output is rounded once: u_out |o|.  Every weight is rounded once to the matrix
              type, bf16 or fp16 (an e4m3 cache: fp16): u_w A, and stands for 2^s with s off by at most
              d = (head_size + 4) 2^-23 S, S = the largest scale log2(e) sum |q k| of the row (sums of the matrix unit are
              taken as truncating), plus 2^-22 of exp2: a relative (d ln 2 + 2^-22), in the numerator and in the sum.
              Sums over L keys in 32 bits: (L / 16 + 32) 2^-23 A twice.  fp16 weights below 2^-22 of the row's largest
              lose bits: L 2^-32 max |v| at most.
  norm        32-bit arithmetic on head_size terms: (head_size + 16) 2^-24 of |x w| r (1 + 1) for the two products of a
              rotation, plus one rounding of the result.
  cache       exact.
"""
import math

import pytest
import torch

from triteia_b200 import _lib, capi, ops

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------------------------------------ plain statements
def plain_codes(x):
    """(value / 2^e rounded to the e4m3 grid, e) of the heads (last axis) of x, in 64 bits."""
    x = x.double()
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    # frexp and not log2, which the device rounds: log2 of 2^k need not be k.  top / 448 is exact where it is a power of two.
    m, e = torch.frexp(top / 448)
    e = torch.where(top > 0, e - (m == 0.5).int(), torch.zeros_like(e)).double().clamp(min=-126)
    r = x / torch.exp2(e)[..., None]
    step = torch.exp2((torch.frexp(r)[1].double() - 1).clamp(min=-6) - 3)
    codes = torch.round(r / step) * step
    return torch.where(fine, codes, float("nan")), e


def quantise(x):
    """(e4m3 codes, exponent bytes) of x, heads on the last axis."""
    codes, e = plain_codes(x)
    return codes.to(torch.float32).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def same(a, b):
    """Equal values, NaN in the same places (heads with an infinity: fp16 overflows in some of the inputs)."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7), b.nan_to_num(7))


def numbers(cache, exps):
    x = cache.double()
    return x if exps is None else x * torch.exp2(exps.double() - 127)[..., None]


def plain_attention(q, keys, values, length, n, scale, causal, window, absent=()):
    """(o, A, S) of n new tokens q [n, heads, size] over keys / values [length, kv heads, size] (64 bits); `absent`: positions
    on pages outside the cache."""
    g = q.shape[1] // keys.shape[1]
    k, v = keys.repeat_interleave(g, 1), values.repeat_interleave(g, 1)
    p = torch.arange(n, device=q.device)[:, None] + (length - n)
    j = torch.arange(length, device=q.device)[None]
    seen = torch.ones(n, length, dtype=torch.bool, device=q.device)
    if causal:
        seen &= j <= p
    if window:
        seen &= j > p - window
    for a in absent:
        seen[:, a] = False
    s = torch.einsum("nhd,lhd->nhl", q.double(), k) * scale
    s = s.masked_fill(~seen[:, None], float("-inf"))
    w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if length else s
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    big = (torch.einsum("nhd,lhd->nhl", q.double().abs(), k.abs()) * seen[:, None]).amax(-1) * abs(scale) * math.log2(math.e) if length else \
        torch.zeros(n, q.shape[1], device=q.device, dtype=torch.float64)
    return torch.einsum("nhl,lhd->nhd", w, v), torch.einsum("nhl,lhd->nhd", w, v.abs()), big


def tolerance(o, A, S, length, dtype, e4m3, size, vmax):
    u_w = 2.0 ** -11 if e4m3 or dtype == torch.float16 else 2.0 ** -8
    d = (size + 4) * 2.0 ** -23 * S[..., None]
    rel = u_w + 2 * (d * math.log(2) + 2.0 ** -22) + 2 * (length / 16 + 32) * 2.0 ** -23
    return U[dtype] * (o.abs() + A * rel) + A * rel + length * 2.0 ** -32 * vmax + (2.0 ** -25 if dtype == torch.float16 else 1e-38)


class Batch:
    """Sequences with shuffled pages; whatever lies at or beyond a sequence's length, and every page that nobody has, is NaN."""

    def __init__(self, seed, lengths, new, heads, kv_heads, size, page, dtype, e4m3, spread=0.0, layout="token"):
        g = gen(seed)
        self.lengths, self.new, self.dtype, self.e4m3 = lengths, new, dtype, e4m3
        used = [-(-n // page) for n in lengths]
        pages, width = sum(used) + 3, max(used + [1])
        order = torch.randperm(pages, generator=g, device="cuda").int()
        self.table = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32, device="cuda")
        kv = [normal(g, pages, page, kv_heads, size, dtype=torch.float32) for _ in range(2)]
        if spread:
            kv = [x * torch.exp2(spread * torch.randn(pages, page, kv_heads, 1, generator=g, device="cuda")) for x in kv]
        kv = [x.to(dtype) for x in kv]
        dead = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        at = 0
        for b, (u, n) in enumerate(zip(used, lengths)):
            self.table[b, :u] = order[at:at + u]
            slots = torch.arange(n, device="cuda")
            dead[order[at:at + u].long()[slots // page], slots % page] = False
            at += u
        if e4m3:
            (self.kc, self.ke), (self.vc, self.ve) = quantise(kv[0]), quantise(kv[1])
            for c in (self.kc, self.vc):
                c.view(torch.uint8)[dead] = 0x7f
            for e in (self.ke, self.ve):
                e[dead] = 255
        else:
            self.kc, self.vc, self.ke, self.ve = kv[0], kv[1], None, None
            for c in (self.kc, self.vc):
                c[dead] = float("nan")
        if layout == "head":      # heads before the tokens of a page
            self.kc, self.vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (self.kc, self.vc))
            if e4m3:
                self.ke, self.ve = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (self.ke, self.ve))
        self.page = page
        self.q = normal(g, sum(new), heads, size, dtype=dtype)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.len = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def tokens(self, b):
        n = self.lengths[b]
        j = torch.arange(n, device="cuda")
        page, place = self.table[b].long()[j // self.page], j % self.page
        e = (None, None) if self.ke is None else (self.ke[page, place], self.ve[page, place])
        return numbers(self.kc[page, place], e[0]), numbers(self.vc[page, place], e[1])

    def call(self, **kw):
        return ops.paged_attention(self.q, self.kc, self.vc, self.table, self.len, self.starts, key_exponents=self.ke,
                                   value_exponents=self.ve, **kw)

    def check(self, out, scale=None, causal=True, window=None):
        size = self.q.shape[2]
        scale = size ** -0.5 if scale is None else scale
        at = 0
        for b, (length, n) in enumerate(zip(self.lengths, self.new)):
            k, v = self.tokens(b)
            o, A, S = plain_attention(self.q[at:at + n], k, v, length, n, scale, causal, window)
            got = out[at:at + n].double()
            assert torch.isfinite(got).all(), f"sequence {b}: not finite"
            vmax = float(v.abs().max()) if length else 0.0
            off = (got - o).abs() - tolerance(o, A, S, length, self.dtype, self.e4m3, size, vmax)
            assert n == 0 or float(off.max()) <= 0, f"sequence {b} ({n} of {length}): {float(off.max())} over the tolerance"
            at += n


DECODE = ([1, 0, 16, 17, 255, 1000, 63, 64, 65], [1] * 9)
CHUNKS = ([5, 40, 300, 0, 129, 64, 77], [5, 3, 130, 0, 1, 64, 76])
SHORT = ([3, 0, 70, 33], [7, 4, 2, 40])            # more new tokens than the cache has: the first see nothing
LONG = ([700, 1500], [300, 515])
LONG_SHORT = ([300, 100, 0], [400, 150, 200])      # the same in calls that the matrix products bound


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kv_heads,size,page", [(8, 2, 128, 16), (4, 4, 64, 16), (6, 2, 128, 24), (5, 1, 64, 128), (40, 2, 128, 7), (3, 3, 128, 64),
                                                      (16, 2, 64, 1)])
@pytest.mark.parametrize("plan", [DECODE, CHUNKS, SHORT, LONG], ids=["decode", "chunks", "short", "long"])
def test_attention(cuda, dtype, e4m3, heads, kv_heads, size, page, plan):
    b = Batch(1, *plan, heads, kv_heads, size, page, dtype, e4m3)
    b.check(b.call())
    if plan is DECODE:
        b.starts = None
        b.check(b.call())


@pytest.mark.parametrize("dtype,e4m3", [(torch.float16, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("causal,window", [(False, None), (True, 1), (True, 16), (True, 100), (True, 5000)])
@pytest.mark.parametrize("plan", [DECODE, CHUNKS, SHORT, LONG, LONG_SHORT], ids=["decode", "chunks", "short", "long", "long-short"])
def test_attention_masks(cuda, dtype, e4m3, causal, window, plan):
    b = Batch(2, *plan, 8, 2, 128, 16, dtype, e4m3)
    b.check(b.call(causal=causal, window=window), causal=causal, window=window)


@pytest.mark.parametrize("dtype,e4m3", [(torch.float16, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (True, 16), (True, 100)])
@pytest.mark.parametrize("size,page", [(128, 8), (64, 40)])
@pytest.mark.parametrize("plan", [CHUNKS, SHORT, LONG], ids=["chunks", "short", "long"])
def test_attention_masks_over_small_pages(cuda, dtype, e4m3, causal, window, size, page, plan):
    b = Batch(17, *plan, 8, 2, size, page, dtype, e4m3)
    b.check(b.call(causal=causal, window=window), causal=causal, window=window)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scale(cuda, scale):
    b = Batch(3, *CHUNKS, 8, 4, 64, 16, torch.float16, False)
    b.check(b.call(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("plan", [DECODE, LONG], ids=["decode", "long"])
def test_attention_over_values_of_very_different_magnitude(cuda, dtype, plan):
    b = Batch(4, *plan, 8, 2, 128, 16, dtype, True, spread=3.0)
    b.check(b.call())


def test_attention_e4m3_tiny_and_large_values(cuda):
    for factor in (2.0 ** -60, 2.0 ** 60):
        b = Batch(5, *DECODE, 8, 2, 64, 16, torch.bfloat16, True)
        shift = round(math.log2(factor))
        alive = b.ve != 255
        b.ve = torch.where(alive, (b.ve.int() + shift).clamp(1, 254), b.ve.int()).to(torch.uint8)
        b.check(b.call())


@pytest.mark.parametrize("new", [1, 20, 130])
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("small", [-20, -40])
def test_attention_to_tiny_values_next_to_large_ones(cuda, new, size, small):
    """Every third token has values 2^`small` times the others' and all of the weight: the large ones of the same tiles must
    not take the small ones' bits (bf16 numbers in an e4m3 cache)."""
    b = Batch(15, [300, 170], [new, new], 8, 2, size, 16, torch.bfloat16, True)
    for i, n in enumerate(b.lengths):
        j = torch.arange(n, device="cuda")
        page, place = b.table[i].long()[j // 16], j % 16
        tiny = j % 3 == 0
        e = b.ve[page, place].int()
        b.ve[page, place] = torch.where(tiny[:, None], e + small, e).to(torch.uint8)
        keys = b.kc[page, place].float()
        keys = torch.where(tiny[:, None, None], keys, torch.full_like(keys, -448.0))
        b.kc.view(torch.uint8)[page, place] = keys.to(torch.float8_e4m3fn).view(torch.uint8)
    b.q = b.q.abs() + 0.25
    b.check(b.call())
    k, v = b.tokens(0)
    o, _, _ = plain_attention(b.q[:new], k, v, 300, new, size ** -0.5, True, None)
    assert float(o.abs().max()) < 2.0 ** -16       # against values of about 1: the case is what it says


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("plan", [DECODE, CHUNKS, LONG], ids=["decode", "chunks", "long"])
def test_attention_strides(cuda, e4m3, plan):
    """Queries inside a fused projection, a cache with the heads outside, a page table inside a wider one, a strided output."""
    b = Batch(6, *plan, 8, 2, 128, 32, torch.bfloat16, e4m3, layout="head")
    T = b.q.shape[0]
    wide = normal(gen(7), T, 13, 128, dtype=torch.bfloat16)
    wide[:, 2:10] = b.q
    b.q = wide[:, 2:10]
    table = torch.full((b.table.shape[0], b.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table
    b.table = table[:, :b.table.shape[1]]
    room = torch.full((8, T, 136), 9.0, dtype=torch.bfloat16, device="cuda")
    out = room.transpose(0, 1)[:, :, :128]
    assert b.call(out=out) is out
    b.check(out)
    assert bool((room[:, :, 128:] == 9).all())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_attention_pages_outside_the_cache_count_as_masked(cuda, e4m3, new):
    length, page = 400, 16
    b = Batch(8, [length, length], [new, new], 8, 2, 128, page, torch.float16, e4m3)
    keep = b.table.clone()
    pages = b.kc.shape[0]
    absent = {1: -1, 7: pages, 12: 1 << 30, 24: -(1 << 31), 0: -5}
    for at, what in absent.items():
        b.table[0, at] = what
    b.table[1, :] = -1                              # nothing of the second sequence is there
    out = b.call()
    b.table = keep
    k, v = b.tokens(0)
    gone = [j for at in absent for j in range(at * page, min((at + 1) * page, length))]
    o, A, S = plain_attention(b.q[:new], k, v, length, new, 128 ** -0.5, True, None, gone)
    got = out[:new].double()
    assert float(((got - o).abs() - tolerance(o, A, S, length, b.dtype, e4m3, 128, float(v.abs().max()))).max()) <= 0
    assert bool((out[new:] == 0).all())


@pytest.mark.parametrize("plan", [CHUNKS, LONG], ids=["chunks", "long"])
def test_attention_leaves_rows_behind_the_last_sequence(cuda, plan):
    b = Batch(9, *plan, 8, 2, 128, 16, torch.float16, False)
    T = b.q.shape[0]
    b.q = torch.cat([b.q, torch.full_like(b.q[:50], float("nan"))])
    out = torch.full((T + 50, 8, 128), 3.0, dtype=torch.float16, device="cuda")
    b.call(out=out)
    b.check(out[:T])
    assert bool((out[T:] == 3).all())


def test_attention_keeps_within_the_batch_whatever_the_starts_say(cuda):
    b = Batch(10, [100, 200, 50], [10, 20, 5], 8, 2, 128, 16, torch.float16, False)
    good = b.call()
    b.starts = torch.tensor([0, 10, 30, 1 << 30], dtype=torch.int32, device="cuda")        # the last one ends with the batch
    assert torch.equal(b.call()[:30], good[:30])
    b.starts = torch.tensor([-9, 10, 4, 35], dtype=torch.int32, device="cuda")             # a sequence that ends before it begins
    assert torch.equal(b.call()[:4], good[:4])
    b.starts = torch.tensor([0, 10, 30, 35], dtype=torch.int32, device="cuda")
    b.len = torch.tensor([1 << 30, -4, 50], dtype=torch.int32, device="cuda")              # beyond the table; below zero
    out = b.call()
    assert bool((out[10:30] == 0).all()) and torch.equal(out[30:], good[30:])


@pytest.mark.parametrize("plan,e4m3", [(DECODE, False), (DECODE, True), (LONG, False), (LONG, True)])
def test_attention_gives_the_same_bits_again_in_graphs_and_on_other_streams(cuda, plan, e4m3):
    b = Batch(11, *plan, 8, 2, 128, 16, torch.bfloat16, e4m3)
    want = b.call().clone()
    c = Batch(12, *plan, 8, 2, 128, 16, torch.bfloat16, e4m3)
    want_c = c.call().clone()
    assert torch.equal(b.call(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = b.call()
    graphs = []
    for x in (b, c):                  # two graphs captured on one stream, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = x.call()
        graphs.append((graph, out))
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(on_side, want) and torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_c)


@pytest.mark.parametrize("plan", [DECODE, CHUNKS, ([900, 40, 2000], [1, 1, 1])], ids=["decode", "chunks", "long-decode"])
def test_attention_calls_side_by_side_on_two_streams(cuda, plan):
    batches = [Batch(70 + i, *plan, 8, 2, 128, 16, torch.float16, i == 1) for i in range(2)]
    want = [b.call().clone() for b in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in batches], [[], []]
    for _ in range(20):
        for i, b in enumerate(batches):
            with torch.cuda.stream(streams[i]):
                got[i].append(b.call())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_attention_refuses_a_workspace_that_is_too_small(cuda):
    b = Batch(20, [5000, 3000], [1, 1], 8, 2, 128, 16, torch.float16, False)
    out = torch.full_like(b.q, 5)
    need = _lib.lib.trb_paged_attention_workspace_bytes(2, 2, 8, 2, 128, 16, b.table.shape[1], 1, 0, 0)
    assert need > 0
    room = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call(workspace, nbytes):
        s = b.kc.stride()
        return _lib.lib.trb_paged_attention(
            _lib.ptr(b.q), _lib.ptr(b.kc), _lib.ptr(b.vc), None, None, _lib.ptr(b.table), _lib.ptr(b.len), None, _lib.ptr(out), 2, 2, 8, 2, 128, 16,
            b.kc.shape[0], b.table.stride(0), b.table.shape[1], b.q.stride(0), b.q.stride(1), out.stride(0), out.stride(1), s[0], s[1], s[2], 0, 0, 0,
            128 ** -0.5, 1, 0, 0, workspace, nbytes, 0, _lib.stream_of(b.q))

    assert call(None, 0) == _lib.ERR_SCRATCH and call(_lib.ptr(room), need - 16) == _lib.ERR_SCRATCH
    assert bool((out == 5).all())
    assert call(_lib.ptr(room), need) == _lib.TRB_OK
    b.check(out)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 9, 260])
def test_attention_in_a_cache_beyond_32_bit_offsets(cuda, e4m3, new):
    """Pages 2^28 elements apart: the last ones begin beyond 2^32 elements."""
    pages, page, kvh, size, stride = 18, 32, 2, 128, 1 << 28
    dtype = torch.float8_e4m3fn if e4m3 else torch.float16
    need = (pages - 1) * stride + page * kvh * size
    room = [torch.empty(need, dtype=dtype, device="cuda") for _ in range(2)]
    small = Batch(13, [pages * page - 40], [new], 4, kvh, size, page, torch.float16, e4m3)
    table = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")[None]
    for r, name in zip(room, ("kc", "vc")):
        view = r.as_strided((pages, page, kvh, size), (stride, kvh * size, size, 1))
        used = small.table.shape[1]
        view.view(torch.uint8 if e4m3 else torch.int16)[table[0, :used].long()] = getattr(small, name).view(torch.uint8 if e4m3 else torch.int16)[small.table[0].long()]
        setattr(small, name, view)
    if e4m3:
        for name in ("ke", "ve"):
            e = torch.full((pages, page, kvh), 255, dtype=torch.uint8, device="cuda")
            e[table[0, :used].long()] = getattr(small, name)[small.table[0].long()]
            setattr(small, name, e)
    small.table = table
    small.check(small.call())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 300])
def test_attention_where_a_stride_says_nothing(cuda, e4m3, new):
    """One key head, one page, one query head, one token: dimensions of one entry, with strides of no use."""
    b = Batch(16, [32], [min(new, 32)], 1, 1, 64, 32, torch.float16, e4m3)
    page = int(b.table[0, 0])
    b.table[0, 0] = 0

    def odd(x):
        return x[page:page + 1].as_strided((1, 32, 1, 64), (7, 64, 5, 1), x[page:page + 1].storage_offset())

    def odd_exps(x):
        return None if x is None else x[page:page + 1].as_strided((1, 32, 1), (3, 1, 9), x[page:page + 1].storage_offset())

    b.kc, b.vc, b.ke, b.ve = odd(b.kc), odd(b.vc), odd_exps(b.ke), odd_exps(b.ve)
    T = b.q.shape[0]
    b.q = b.q.as_strided((T, 1, 64), (11 if T == 1 else 64, 13, 1))
    b.check(b.call())
    if new == 1:
        b.starts = None
        b.check(b.call())
    slots = torch.arange(32, device="cuda")
    k, v = ops.cache_read(b.kc, b.vc, slots, b.ke, b.ve, dtype=torch.float16)
    again = (b.kc.clone(), b.vc.clone(), None if b.ke is None else b.ke.clone(), None if b.ve is None else b.ve.clone())
    ops.cache_write(k.as_strided((32, 1, 64), (64, 3, 1)), v, again[0], again[1], slots, again[2], again[3])
    assert torch.equal(torch.stack(ops.cache_read(again[0], again[1], slots, again[2], again[3], dtype=torch.float16)), torch.stack((k, v)))


@pytest.mark.parametrize("new", [1, 3, 200])
def test_attention_without_pages(cuda, new):
    """Sequences whose table has no columns: nothing is seen."""
    kc, vc, _, _ = ops.new_cache(2, 16, 2, 64)
    q = normal(gen(17), 2 * new, 4, 64)
    out = ops.paged_attention(q, kc, vc, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.full((2,), 50, dtype=torch.int32, device="cuda"),
                              torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda"))
    assert bool((out == 0).all())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(64, 1), (96, 1), (200, 1), (17, 1)])
def test_attention_of_many_heads_over_one(cuda, e4m3, heads, kv_heads):
    for plan in (([100, 0, 33], [1, 1, 1]), ([100, 40], [7, 12]), ([200, 300], [30, 1])):
        b = Batch(18, *plan, heads, kv_heads, 64, 16, torch.bfloat16, e4m3)
        b.check(b.call())
        if sum(plan[1]) == len(plan[1]):
            b.starts = None
            b.check(b.call())


def test_attention_of_more_sequences_than_a_warp_has_lanes(cuda):
    lengths = [(37 * i) % 150 for i in range(70)]
    for new in ([1] * 70, [(i % 5) * 3 for i in range(70)]):
        b = Batch(19, lengths, new, 8, 2, 64, 16, torch.float16, False)
        b.check(b.call())
        if new == [1] * 70:
            b.starts = None
            b.check(b.call())


@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_far_into_a_document(cuda, e4m3):
    b = Batch(14, [100_003, 31], [1, 1], 8, 2, 128, 64, torch.bfloat16, e4m3)
    b.check(b.call())


@pytest.mark.parametrize("dtype,e4m3", [(torch.float16, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (True, 100)])
@pytest.mark.parametrize("heads,kv_heads,size,page", [(8, 2, 128, 16), (40, 20, 128, 24), (80, 40, 64, 64)])
@pytest.mark.parametrize("lengths,new", [([3000], [60]), ([2900, 0, 1200], [70, 0, 40]), ([2500, 200], [64, 200]), ([1700], [300])],
                         ids=["one", "three", "uneven", "wide"])
def test_attention_of_few_tokens_over_many(cuda, dtype, e4m3, causal, window, heads, kv_heads, size, page, lengths, new):
    b = Batch(16, lengths, new, heads, kv_heads, size, page, dtype, e4m3)
    out = b.call(causal=causal, window=window)
    b.check(out, causal=causal, window=window)
    for _ in range(3):
        assert same(out, b.call(causal=causal, window=window))


# ------------------------------------------------------------------------------------------------ cache
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("T,heads,size,page", [(1, 1, 128, 16), (7, 8, 64, 16), (333, 5, 80, 24), (61, 40, 128, 1), (19, 2, 256, 128), (2000, 3, 8, 32), (5, 150, 32, 16),
                                                    (3, 700, 8, 16), (700, 33, 16, 16)])
def test_cache_write_and_read(cuda, dtype, quantised, T, heads, size, page):
    g = gen(20)
    pages = -(-T // page) + 2
    kc, vc, ke, ve = ops.new_cache(pages, page, heads, size, dtype, quantised)
    fused = normal(g, T, 3 * heads, size, dtype=torch.float32)
    fused = (fused * torch.exp2(4 * torch.randn(T, 3 * heads, 1, generator=g, device="cuda"))).to(dtype)
    key, value = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].clone()
    slots[T // 2] = -1
    if T > 4:
        slots[1] = pages * page
    keep = (slots >= 0) & (slots < pages * page)
    before = kc.view(torch.uint8).clone()
    ops.cache_write(key, value, kc, vc, slots, ke, ve)
    rk, rv = ops.cache_read(kc, vc, slots, ke, ve, dtype=dtype)
    for x, cache, exps, back in ((key, kc, ke, rk), (value, vc, ve, rv)):
        flat = cache.flatten(0, 1)
        if quantised:
            codes, e = plain_codes(x)
            assert same(flat.view(torch.uint8)[slots[keep]].view(torch.float8_e4m3fn).double(), codes[keep])
            assert torch.equal(exps.flatten(0, 1)[slots[keep]].double() - 127, e[keep])
            want = (codes * torch.exp2(e)[..., None]).to(dtype)
        else:
            assert same(flat[slots[keep]], x[keep])
            want = x
        assert same(back[keep], want[keep]) and bool((back[~keep] == 0).all())
    others = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    others[slots[keep]] = False
    assert torch.equal(kc.view(torch.uint8).flatten(0, 1)[others], before.flatten(0, 1)[others])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_cache_quantises_borders_ties_and_what_is_no_number(cuda, dtype):
    big = float(torch.finfo(dtype).max)
    tiny = float(torch.finfo(dtype).tiny)
    rows = torch.zeros(14, 1, 16, dtype=torch.float32)
    rows[1, 0, 0] = 448
    rows[2, 0, :2] = torch.tensor([449.0, 1.0]) if dtype == torch.float16 else torch.tensor([450.0, 1.0])
    rows[3, 0] = torch.tensor([1.0, 1.0625, 1.1875, 1.3125, 17, 19, 21, 23, 0.01, -1.0625, -17, 256, 240, 248, 2 ** -7, 3 * 2 ** -8])
    rows[4, 0, :3] = torch.tensor([float("inf"), 2.0, -3.0])
    rows[5, 0, :3] = torch.tensor([float("nan"), 2.0, -3.0])
    rows[6, 0] = float("-inf")
    rows[7, 0] = float("nan")
    rows[8, 0, :2] = torch.tensor([big, 1.0])
    rows[9, 0, 3] = tiny
    rows[10, 0, 3] = -tiny / 8
    rows[11, 0] = torch.linspace(-2, 2, 16)
    rows[12, 0] = -0.0
    rows[13, 0] = 2.0 ** torch.arange(-8, 8)
    x = rows.to(dtype).cuda()
    kc, vc, ke, ve = ops.new_cache(1, 16, 1, 16, dtype, True)
    slots = torch.arange(14, device="cuda")
    ops.cache_write(x, x, kc, vc, slots, ke, ve)
    codes, e = plain_codes(x)
    got = kc[0, :14].double()
    assert same(got, codes)
    assert torch.equal(ke[0, :14].double() - 127, e) and torch.equal(ke, ve)
    back, _ = ops.cache_read(kc, vc, slots, ke, ve, dtype=dtype)
    want = (codes * torch.exp2(e)[..., None]).to(dtype)
    assert same(back, want)


@pytest.mark.parametrize("quantised", [False, True])
def test_cache_beyond_32_bit_offsets_and_permuted(cuda, quantised):
    pages, page, heads, size, stride = 18, 16, 2, 128, 1 << 28
    dtype = torch.float8_e4m3fn if quantised else torch.float16
    need = (pages - 1) * stride + page * heads * size
    kc, vc = (torch.empty(need, dtype=dtype, device="cuda").as_strided((pages, page, heads, size), (stride, size, page * size, 1)) for _ in range(2))
    ke = ve = None
    if quantised:
        ke, ve = (torch.zeros(heads, pages, page, dtype=torch.uint8, device="cuda").permute(1, 2, 0) for _ in range(2))
    x = normal(gen(21), 2, pages * page, heads, size)
    slots = torch.randperm(pages * page, generator=gen(22), device="cuda")
    ops.cache_write(x[0], x[1], kc, vc, slots, ke, ve)
    rk, rv = ops.cache_read(kc, vc, slots, ke, ve, dtype=torch.float16)
    for a, b in ((x[0], rk), (x[1], rv)):
        if quantised:
            codes, e = plain_codes(a)
            a = (codes * torch.exp2(e)[..., None]).half()
        assert torch.equal(a, b)


def test_cache_calls_with_no_tokens(cuda):
    kc, vc, _, _ = ops.new_cache(2, 16, 2, 64)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    ops.cache_write(torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda"), torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda"), kc, vc, none)
    assert ops.cache_read(kc, vc, none)[0].shape == (0, 2, 64)
    assert ops.paged_attention(torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda"), kc, vc, torch.zeros(0, 3, dtype=torch.int32, device="cuda"),
                               torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


# ------------------------------------------------------------------------------------------------ norm and rotation
def plain_norm_rotary(pos, x, size, table, neox, weight, eps):
    T, rot = x.shape[0], table.shape[1]
    x = x.double().reshape(T, -1, size)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    row = table.double()[pos][:, None]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    out, mag = y.clone(), y.abs()
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    mag[..., a], mag[..., b] = (y[..., a] * c).abs() + (y[..., b] * s).abs(), (y[..., b] * c).abs() + (y[..., a] * s).abs()
    return out.reshape(T, -1), mag.reshape(T, -1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("T,heads,kv_heads,size,rot", [(1, 1, 1, 128, 128), (7, 32, 8, 128, 128), (130, 5, 3, 64, 32), (33, 4, 2, 80, 80), (9, 3, 1, 80, 20),
                                                       (5, 2, 2, 256, 64), (3, 9, 1, 8, 8), (600, 40, 40, 128, 64), (4, 2, 0, 96, 0), (11, 2, 1, 24, 22)])
def test_qk_norm_rotary(cuda, dtype, neox, wide, T, heads, kv_heads, size, rot):
    g = gen(30)
    fused = normal(g, T, (heads + 2 * kv_heads) * size + 8, dtype=dtype) * 3
    q, k = fused[:, :heads * size], fused[:, heads * size:(heads + kv_heads) * size] if kv_heads else None
    angle = torch.rand(50, max(rot // 2, 0), generator=g, device="cuda") * 6.28
    table = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32 if wide else dtype)
    pos = torch.randint(0, 50, (T,), generator=g, device="cuda")
    qw = (1 + 0.2 * normal(g, size)).to(dtype)
    kw = None if T == 7 else (1 + 0.2 * normal(g, size)).to(dtype)
    skip = T // 2 if T > 2 else None
    if skip is not None:
        pos[skip] = 50 if T % 2 else -1
    before = fused.clone()
    qo, ko = torch.full_like(before[:, :heads * size], 5), None if k is None else torch.full_like(k, 5).contiguous()
    capi.qk_norm_rotary_embedding(pos, q, k, size, table, neox, qw, kw, 1e-5, qo, ko)
    assert torch.equal(fused, before)
    live = torch.ones(T, dtype=torch.bool, device="cuda")
    if skip is not None:
        live[skip] = False
        assert bool((qo[skip] == 5).all()) and (ko is None or bool((ko[skip] == 5).all()))
    for x, w, got in ((q, qw, qo), (k, kw, ko)):
        if x is None:
            continue
        want, mag = plain_norm_rotary(pos.clamp(0, 49), x, size, table, neox, w, 1e-5)
        u = U[dtype]
        tol = u * want.abs() + (1 + u) * (size + 16) * 2.0 ** -24 * mag + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert float(((got.double() - want).abs() - tol)[live].max()) <= 0
    capi.qk_norm_rotary_embedding(pos, q, k, size, table, neox, qw, kw, 1e-5)          # in place: the same values
    assert torch.equal(q[live], qo[live]) and (k is None or torch.equal(k[live], ko[live]))
    rest = torch.ones(fused.shape[1], dtype=torch.bool, device="cuda")
    rest[:(heads + kv_heads) * size] = False
    assert torch.equal(fused[:, rest], before[:, rest])
    if skip is not None:
        assert torch.equal(fused[skip], before[skip])


def test_qk_norm_of_zeros_and_of_three_dimensions(cuda):
    table = torch.cat([torch.ones(4, 32), torch.zeros(4, 32)], 1).half().cuda()
    q = torch.zeros(2, 3, 128, dtype=torch.float16, device="cuda")
    q[1, 2] = 2
    k = q[..., :64].contiguous()
    capi.qk_norm_rotary_embedding(torch.zeros(6, dtype=torch.int64, device="cuda"), q, k, 64, table, True, eps=0.0)
    assert bool((q[1, 2] == 1).all()) and bool((k[1, 2] == 1).all())
    assert torch.isnan(q[0]).all()          # 0 / sqrt(0): without an eps a head of zeros has no norm


def test_refusals_on_the_device(cuda):
    b = Batch(40, [20, 30], [1, 1], 4, 2, 64, 16, torch.float16, False)
    for spoil, what in [
        (dict(lengths=b.len.long()), "lengths"), (dict(lengths=b.len[:1]), "lengths"), (dict(query_starts=b.starts[:2]), "query_starts"),
        (dict(page_table=b.table.long()), "page_table"), (dict(page_table=b.table[:1], lengths=b.len[:1]), "query_starts is needed"),
        (dict(window=0), "window"), (dict(window=3, causal=False), "window"), (dict(query=b.q[:, :3]), "do not go with"),
        (dict(query=b.q.bfloat16()), "the cache holds"), (dict(query=b.q[..., :32]), "do not go with"), (dict(out=b.q.float()), "out"),
        (dict(page_table=b.table.cpu()), "page_table"), (dict(lengths=b.len.cpu()), "lengths"), (dict(key_cache=b.kc.cpu(), value_cache=b.vc.cpu()), "the cache must be on"),
    ]:
        a = dict(query=b.q, key_cache=b.kc, value_cache=b.vc, page_table=b.table, lengths=b.len, query_starts=None) | spoil
        with pytest.raises(RuntimeError, match=what):
            ops.paged_attention(**a)
    with pytest.raises(RuntimeError, match="slots"):
        ops.cache_write(b.kc[0], b.vc[0], b.kc, b.vc, torch.zeros(16, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="slots"):
        ops.cache_write(b.kc[0], b.vc[0], b.kc, b.vc, torch.zeros(15, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="No suitable kernel"):
        ops.cache_read(b.kc, b.vc, torch.zeros(1, dtype=torch.int64, device="cuda"), dtype=torch.float32)
    pos, table = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    q = b.q.view(2, 256)
    for spoil, what in [(dict(positions=pos.int()), "positions"), (dict(positions=pos[:1]), "positions"), (dict(key=q[:1]), "key"),
                        (dict(cos_sin_cache=table.double()), "cos_sin_cache"), (dict(query_weight=table[0, :32]), "query_weight"),
                        (dict(head_size=48), "query must be"), (dict(cos_sin_cache=torch.zeros(4, 128, dtype=torch.float16, device="cuda")), "No suitable kernel"),
                        (dict(key=q.bfloat16()), "key must have")]:
        a = dict(positions=pos, query=q, key=q.clone(), head_size=64, cos_sin_cache=table, is_neox=True) | spoil
        with pytest.raises(RuntimeError, match=what):
            capi.qk_norm_rotary_embedding(**a)


@pytest.mark.parametrize("quantised", [False, True])
def test_a_prompt_in_chunks_and_then_token_by_token(cuda, quantised):
    """Norm and rotation, cache write and attention as a decoder layer uses them: two chunks and three single tokens of two
    sequences, every step against attention over the whole history in 64 bits."""
    heads, kv_heads, size, page, dtype = 8, 2, 128, 16, torch.bfloat16
    g = gen(50)
    steps = [[70, 33], [40, 100], [1, 1], [1, 1], [1, 1]]
    total = [sum(s[b] for s in steps) for b in range(2)]
    pages = [-(-t // page) for t in total]
    table = torch.full((2, max(pages)), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(sum(pages), generator=g, device="cuda").int()
    table[0, :pages[0]], table[1, :pages[1]] = order[:pages[0]], order[pages[0]:]
    kc, vc, ke, ve = ops.new_cache(sum(pages), page, kv_heads, size, dtype, quantised)
    angle = torch.outer(torch.arange(300, device="cuda").double(), 10000.0 ** (-torch.arange(0, size, 2, device="cuda").double() / size))
    rope = torch.cat([angle.cos(), angle.sin()], 1).float()
    qw, kw = (1 + 0.1 * normal(g, 2, size, dtype=torch.float32)).to(dtype)
    done, history = [0, 0], [[], []]
    for step in steps:
        T = sum(step)
        fused = normal(g, T, (heads + 2 * kv_heads) * size, dtype=dtype)
        q, k, v = fused.split([heads * size, kv_heads * size, kv_heads * size], 1)
        pos = torch.cat([torch.arange(done[b], done[b] + step[b], device="cuda") for b in range(2)])
        seq = torch.cat([torch.full((step[b],), b, device="cuda") for b in range(2)])
        slots = table[seq, pos // page].long() * page + pos % page
        capi.qk_norm_rotary_embedding(pos, q, k, size, rope, True, qw, kw)
        k3, v3 = k.unflatten(1, (kv_heads, size)), v.unflatten(1, (kv_heads, size))
        ops.cache_write(k3, v3, kc, vc, slots, ke, ve)
        done = [done[b] + step[b] for b in range(2)]
        starts = torch.tensor([0, step[0], T], dtype=torch.int32, device="cuda") if T > 2 else None
        q3 = q.unflatten(1, (heads, size))
        out = ops.paged_attention(q3, kc, vc, table, torch.tensor(done, dtype=torch.int32, device="cuda"), starts, key_exponents=ke, value_exponents=ve)
        at = 0
        for b in range(2):
            n = step[b]
            new = []
            for x in (k3, v3):
                x = x[at:at + n].double()
                if quantised:
                    codes, e = plain_codes(x)
                    x = codes * torch.exp2(e)[..., None]
                new.append(x)
            history[b].append(new)
            keys, values = (torch.cat([h[i] for h in history[b]]) for i in range(2))
            o, A, S = plain_attention(q3[at:at + n], keys, values, done[b], n, size ** -0.5, True, None)
            off = (out[at:at + n].double() - o).abs() - tolerance(o, A, S, done[b], dtype, quantised, size, float(values.abs().max()))
            assert float(off.max()) <= 0
            at += n
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("neox", [True, False])
def test_rotation_without_a_norm(cuda, neox):
    g = gen(31)
    fused = normal(g, 37, 6 * 64 + 8)
    q, k = fused[:, :256], fused[:, 256:384]
    angle = torch.rand(50, 24, generator=g, device="cuda") * 6.28
    table = torch.cat([angle.cos(), angle.sin()], 1).half()
    pos = torch.randint(0, 50, (37,), generator=g, device="cuda")
    w = (1 + 0.2 * normal(g, 64)).half()
    for weight in (None, w):
        qo, ko = torch.empty_like(q).contiguous(), torch.empty_like(k).contiguous()
        capi.qk_norm_rotary_embedding(pos, q, k, 64, table, neox, weight, weight, None, qo, ko)
        for x, got in ((q, qo), (k, ko)):
            # the plain statement without its norm: scale the input so that the norm is one, and back
            y = x.double().reshape(37, -1, 64)
            n = (y.square().mean(-1, keepdim=True)).sqrt()
            want, mag = plain_norm_rotary(pos, x, 64, table, neox, weight, 0.0)
            want, mag = want * n.expand(-1, -1, 64).reshape(37, -1), mag * n.expand(-1, -1, 64).reshape(37, -1)
            tol = U[torch.float16] * want.abs() + (1 + U[torch.float16]) * 80 * 2.0 ** -24 * mag + 2.0 ** -25
            assert float(((got.double() - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("quantised,qk_norm", [(False, False), (True, True)])
def test_delta_attention_block(cuda, quantised, qk_norm):
    """The module runs its operators in order: a chunk of two sequences of different models and then a token of each, against the
    same operators called one by one on a cache of their own and, between the projections, plain statements in 64 bits."""
    from triteia_b200.nn import delta_attention

    hidden, heads, kv_heads, size, D, page = 512, 4, 2, 128, 3, 16
    m = delta_attention(hidden, heads, kv_heads, size, D, max_position=128, groupsize=128, qk_norm=qk_norm).to(cuda)
    g = gen(60)
    for name, k, n in (("qkv", hidden, 8 * size), ("o", heads * size, hidden)):
        q, meta, s = ops.random_packed_deltas(D, k, n, groupsize=128, device=cuda, seed=1, scale_lo=0.002, scale_hi=0.004)
        getattr(m, name + "_qweight").copy_(q), getattr(m, name + "_meta").copy_(meta), getattr(m, name + "_scale").copy_(s)
        getattr(m, name + "_weight").copy_(normal(g, n, k) * k ** -0.5)
    angle = torch.outer(torch.arange(128, device="cuda").double(), 10000.0 ** (-torch.arange(0, size, 2, device="cuda").double() / size))
    m.cos_sin_cache.copy_(torch.cat([angle.cos(), angle.sin()], 1))
    cache, own = (ops.new_cache(6, page, kv_heads, size, torch.float16, quantised) for _ in range(2))
    table = torch.tensor([[4, 1, -1], [0, 3, 5]], dtype=torch.int32, device="cuda")
    done, model = [0, 0], [2, -1]
    history = [[], []]
    for step in ([20, 33], [1, 1]):
        T = sum(step)
        x = normal(g, T, hidden)
        pos = torch.cat([torch.arange(done[b], done[b] + step[b], device="cuda") for b in range(2)])
        seq = torch.cat([torch.full((step[b],), b, device="cuda") for b in range(2)])
        slots = table[seq, pos // page].long() * page + pos % page
        idx = torch.tensor(model, dtype=torch.int32, device="cuda")[seq]
        done = [done[b] + step[b] for b in range(2)]
        lengths = torch.tensor(done, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, step[0], T], dtype=torch.int32, device="cuda") if T > 2 else None
        y = m(x, idx, pos, slots, cache, table, lengths, starts)
        qkv = ops.sbmm_4bit_2_4_native(m.qkv_qweight, x, m.qkv_meta, m.qkv_scale, idx, base_weight=m.qkv_weight)
        q, k, v = qkv.split([heads * size, kv_heads * size, kv_heads * size], 1)
        capi.qk_norm_rotary_embedding(pos, q, k, size, m.cos_sin_cache, True, m.query_norm, m.key_norm, 1e-6 if qk_norm else None)
        q, k, v = (t.unflatten(1, (-1, size)) for t in (q, k, v))
        ops.cache_write(k, v, own[0], own[1], slots, own[2], own[3])
        out = ops.paged_attention(q, own[0], own[1], table, lengths, starts, key_exponents=own[2], value_exponents=own[3])
        assert torch.equal(y, ops.sbmm_4bit_2_4_native(m.o_qweight, out.flatten(1), m.o_meta, m.o_scale, idx, base_weight=m.o_weight))
        at = 0
        for b in range(2):
            n = step[b]
            new = [t[at:at + n].double() for t in (k, v)]
            if quantised:
                new = [c * torch.exp2(e)[..., None] for c, e in map(plain_codes, new)]
            history[b].append(new)
            keys, values = (torch.cat([h[i] for h in history[b]]) for i in range(2))
            o, A, S = plain_attention(q[at:at + n], keys, values, done[b], n, size ** -0.5, True, None)
            assert float(((out[at:at + n].double() - o).abs() - tolerance(o, A, S, done[b], torch.float16, quantised, size, float(values.abs().max()))).max()) <= 0
            at += n


def test_delta_attention_refuses_heads_that_do_not_divide(cuda):
    from triteia_b200.nn import delta_attention

    with pytest.raises(ValueError, match="key heads"):
        delta_attention(512, 5, 2, 128, 1, 16)
