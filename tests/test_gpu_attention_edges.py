"""GPU: attention where a cache, a mask or a batch is unusual.  Statements and tolerances as in test_gpu_attention.py."""
import math

import pytest
import torch

from test_gpu_attention import LONG_SHORT, SHORT, Batch, gen, normal, plain_attention, tolerance
from triteia_b200 import capi, ops

pytestmark = pytest.mark.gpu


def check(b, out, scale=None, vmax=None, causal=True, window=None):
    """Batch.check with the largest value that has weight (vmax) given: one that has none must not widen the tolerance."""
    size, at = b.q.shape[2], 0
    scale = size ** -0.5 if scale is None else scale
    for i, (length, n) in enumerate(zip(b.lengths, b.new)):
        k, v = b.tokens(i)
        o, A, S = plain_attention(b.q[at:at + n], k, v, length, n, scale, causal, window)
        got = out[at:at + n].double()
        assert torch.isfinite(got).all(), f"sequence {i}: not finite"
        most = float(v.abs().max()) if vmax is None else vmax
        off = (got - o).abs() - tolerance(o, A, S, length, b.dtype, b.e4m3, size, most)
        assert float(off.max()) <= 0, f"sequence {i} ({n} of {length}): {float(off.max())} over the tolerance"
        at += n


def places(b, i, positions):
    j = torch.as_tensor(positions, device="cuda")
    return b.table[i].long()[j // b.page], j % b.page


# (new tokens, page): the warps split the tokens; the warps split the rows; tensor memory
KERNELS = [(1, 16), (40, 24), (40, 16), (130, 16)]


@pytest.mark.parametrize("new,page", KERNELS)
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("magnitude,ahead", [(-5, 10), (-10, 10), (-14, 7), (-14, 10), (-16, 0), (-20, 0), (-20, 10), (-30, 0), (-60, 3), (20, 5)])
@pytest.mark.parametrize("zeros", ["one", "run", "last"])
def test_value_heads_of_zeros_in_an_e4m3_cache(cuda, new, page, size, magnitude, ahead, zeros):
    """A visible token whose value head is zero has the exponent byte 127, whatever the other values' magnitude 2^`magnitude`:
    it takes its share of the weight and none of the others' bits.  Its score is about `ahead` above the others'."""
    b = Batch(80, [300, 700], [new, new], 8, 2, size, page, torch.bfloat16, True)
    b.q[..., 0] = 4
    for i, n in enumerate(b.lengths):
        page_, place = places(b, i, range(n))
        b.kc.view(torch.uint8)[page_, place, :, 0] = 0
        b.ve[page_, place] = (b.ve[page_, place].int() + magnitude).to(torch.uint8)
        page_, place = places(b, i, {"one": [5], "run": range(0, 270), "last": [n - 20, n - 1]}[zeros])
        b.kc.view(torch.uint8)[page_, place] = 0
        b.kc[page_, place, :, 0] = torch.tensor(ahead * size ** 0.5 / 4, device="cuda").to(torch.float8_e4m3fn)
        b.ke[page_, place] = 127
        b.vc.view(torch.uint8)[page_, place] = 0
        b.vc.view(torch.uint8)[page_, place, :, ::3] = 0x80            # -0
        b.ve[page_, place] = 127
    check(b, b.call())
    if new == 1:
        b.starts = None
        check(b, b.call())


@pytest.mark.parametrize("new,page", KERNELS)
def test_one_key_head_has_no_values_at_all(cuda, new, page):
    b = Batch(81, [300, 2100, 17], [new, new, 5], 8, 2, 128, page, torch.float16, True)
    for i, n in enumerate(b.lengths):
        page_, place = places(b, i, range(n))
        b.vc.view(torch.uint8)[page_, place, 1] = 0
        b.ve[page_, place, 1] = 127
        b.ve[page_, place, 0] -= 9
    out = b.call()
    check(b, out)
    assert bool((out[:, 4:] == 0).all())


@pytest.mark.parametrize("new,page", KERNELS)
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("small", [-20, -40])
def test_tiny_values_with_all_the_weight(cuda, new, page, size, small):
    """Every third token has values 2^`small` times the others' and all of the weight (the others' scores are hundreds below),
    so that only the tiny ones' magnitude may enter the tolerance."""
    b = Batch(82, [300, 170], [new, new], 8, 2, size, page, torch.bfloat16, True)
    vmax = 0.0
    for i, n in enumerate(b.lengths):
        page_, place = places(b, i, range(n))
        tiny = torch.arange(n, device="cuda") % 3 == 0
        e = b.ve[page_, place].int()
        b.ve[page_, place] = torch.where(tiny[:, None], e + small, e).to(torch.uint8)
        keys = b.kc[page_, place].float()
        keys = torch.where(tiny[:, None, None], keys, torch.full_like(keys, -448.0))
        b.kc.view(torch.uint8)[page_, place] = keys.to(torch.float8_e4m3fn).view(torch.uint8)
        vmax = max(vmax, float(b.tokens(i)[1][tiny].abs().max()))
    b.q = b.q.abs() + 0.25
    out = b.call()
    check(b, out, vmax=vmax)
    with pytest.raises(AssertionError):
        check(b, torch.zeros_like(out), vmax=vmax)


@pytest.mark.parametrize("new,page", KERNELS)
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("larger", [12, 17, 24, 30, 100])
@pytest.mark.parametrize("where", ["hidden", "orthogonal"])
def test_a_key_that_dwarfs_its_neighbours(cuda, new, page, size, larger, where):
    """One key 2^`larger` times its neighbours' takes no bits of their scores: rows that do not see it, or are orthogonal to it."""
    b = Batch(83, [300, 2100], [new, new], 8, 2, size, page, torch.bfloat16, True)
    for i, n in enumerate(b.lengths):
        if where == "hidden":
            page_, place = places(b, i, [n - 1])
        else:
            page_, place = places(b, i, [n - 30, 3])
            b.kc.view(torch.uint8)[page_, place, :, 1:] = 0
            b.kc[page_, place, :, 0] = torch.tensor(300.0, device="cuda").to(torch.float8_e4m3fn)
        b.ke[page_, place] += larger
    if where == "orthogonal":
        b.q[..., 0] = 0
    out = b.call()
    if where == "hidden":                      # the last row of each sequence sees the large key: its scores may be anything
        b.new = [new - 1, new - 1]
        keep = torch.ones(2 * new, dtype=torch.bool, device="cuda")
        keep[[new - 1, 2 * new - 1]] = False
        b.q, out = b.q[keep], out[keep]
        for i in range(2):
            b.lengths[i] -= 1
        if new == 1:
            return
    check(b, out)


@pytest.mark.parametrize("new,page", KERNELS)
@pytest.mark.parametrize("small", [-16, -24, -60])
def test_key_heads_of_zeros_among_small_keys(cuda, new, page, small):
    """A key head of zeros has the exponent byte 127 and a score of zero; the other keys, 2^`small`, keep their bits."""
    b = Batch(84, [300, 700], [new, new], 8, 2, 128, page, torch.bfloat16, True)
    for i, n in enumerate(b.lengths):
        page_, place = places(b, i, range(n))
        b.ke[page_, place] = (b.ke[page_, place].int() + small).to(torch.uint8)
        page_, place = places(b, i, range(7, n, 50))
        b.kc.view(torch.uint8)[page_, place] = 0
        b.ke[page_, place] = 127
    scale = 128 ** -0.5 * 2.0 ** -small
    check(b, b.call(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype,e4m3", [(torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 40, 2 ** 31 - 300, 1 << 20])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("plan", [SHORT, LONG_SHORT, ([3], [7]), ([5, 300], [1, 1])], ids=["short", "long-short", "one", "single"])
def test_windows_that_hide_nothing(cuda, dtype, e4m3, window, page, plan):
    """Any window as long as the sequences or longer, also with more new tokens than the cache has."""
    b = Batch(85, *plan, 8, 2, 128, page, dtype, e4m3)
    out = b.call(window=window)
    b.check(out)
    assert torch.equal(out, b.call())


def spoiled(shape, dtype):
    """Leaves a block of NaN of this size to the allocator."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    x = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    del x


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,new,front,behind", [
    ([300, 170], [40, 130], 0, 70), ([300, 170], [40, 130], 9, 3), ([0, 0], [0, 0], 0, 50), ([40, 70], [2, 1], 0, 29), ([4000, 70], [2, 1], 2, 29),
    ([5000], [1], 0, 1), ([100], [1], 3, 500), ([4000, 9], [64, 3], 5, 700), ([300, 170], [40, 130], 0, 0)])
@pytest.mark.parametrize("page", [16, 24])
def test_rows_of_no_sequence_are_zero_in_a_new_output(cuda, e4m3, lengths, new, front, behind, page):
    b = Batch(86, lengths, new, 8, 2, 128, page, torch.float16, e4m3)
    T = sum(new)
    q = torch.full((front + T + behind, 8, 128), float("nan"), dtype=torch.float16, device="cuda")
    q[front:front + T] = b.q
    b.q, b.starts = q, b.starts + front
    spoiled(q.shape, q.dtype)
    out = b.call()
    assert bool((out[:front] == 0).all()) and bool((out[front + T:] == 0).all())
    given = torch.full_like(q, 3)
    b.call(out=given)
    assert bool((given[:front] == 3).all()) and bool((given[front + T:] == 3).all()) and torch.equal(given[front:front + T], out[front:front + T])
    b.q = q[front:front + T]
    b.check(out[front:front + T])


def test_a_batch_without_sequences_is_all_padding(cuda):
    kc, vc, _, _ = ops.new_cache(2, 16, 2, 64)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    q = torch.full((5000, 4, 64), float("nan"), dtype=torch.float16, device="cuda")
    spoiled(q.shape, q.dtype)
    for width in (0, 3):
        out = ops.paged_attention(q, kc, vc, none.new_zeros(0, width), none, none.new_zeros(1))
        assert bool((out == 0).all())
    given = torch.full_like(q, 3)
    ops.paged_attention(q, kc, vc, none.new_zeros(0, 3), none, none.new_zeros(1), out=given)
    assert bool((given == 3).all())


def test_delta_attention_of_a_padded_batch(cuda):
    """Padding tokens behind the last sequence (slot -1, position -1): the live rows are those of the batch without them, and the
    output projection gets zeros for the others."""
    from triteia_b200.nn import delta_attention

    hidden, heads, kv_heads, size, page = 512, 4, 2, 128, 16
    m = delta_attention(hidden, heads, kv_heads, size, 2, max_position=128, groupsize=128).to(cuda)
    g = gen(87)
    for name, k, n in (("qkv", hidden, 8 * size), ("o", heads * size, hidden)):
        q, meta, s = ops.random_packed_deltas(2, k, n, groupsize=128, device=cuda, seed=1, scale_lo=0.002, scale_hi=0.004)
        getattr(m, name + "_qweight").copy_(q), getattr(m, name + "_meta").copy_(meta), getattr(m, name + "_scale").copy_(s)
        getattr(m, name + "_weight").copy_(normal(g, n, k) * k ** -0.5)
    angle = torch.outer(torch.arange(128, device="cuda").double(), 10000.0 ** (-torch.arange(0, size, 2, device="cuda").double() / size))
    m.cos_sin_cache.copy_(torch.cat([angle.cos(), angle.sin()], 1))
    table = torch.tensor([[4, 1, -1], [0, 3, 5]], dtype=torch.int32, device="cuda")
    new, T, pad = [20, 33], 53, 11
    x = normal(g, T + pad, hidden)
    pos = torch.cat([torch.arange(n, device="cuda") for n in new] + [torch.full((pad,), -1, device="cuda")])
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(new)])
    slots = torch.cat([table[seq, pos[:T] // page].long() * page + pos[:T] % page, torch.full((pad,), -1, device="cuda")])
    idx = torch.cat([torch.tensor([1, -1], dtype=torch.int32, device="cuda")[seq], torch.full((pad,), -1, dtype=torch.int32, device="cuda")])
    lengths, starts = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (new, [0, 20, 53]))
    outs = []
    for rows in (T + pad, T):
        cache = ops.new_cache(6, page, kv_heads, size, torch.float16, False)
        spoiled((rows, heads, size), torch.float16)
        outs.append(m(x[:rows], idx[:rows], pos[:rows], slots[:rows], cache, table, lengths, starts))
    assert torch.equal(outs[0][:T], outs[1])
    assert bool((outs[0][T:] == 0).all())


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_prompt_takes_no_memory_but_its_output(cuda, e4m3):
    b = Batch(88, [1500, 900], [700, 900], 8, 2, 128, 16, torch.float16, e4m3)
    b.call()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = b.call()
    assert torch.cuda.max_memory_allocated() - before == out.untyped_storage().nbytes()


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("rot", [16, 24, 20, 0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rotation_alone_passes_on_what_it_does_not_turn(cuda, neox, rot, dtype):
    """Sizes behind rot_dim come out as they are, infinities and NaN too, and reach no other size."""
    g = gen(90)
    q = normal(g, 9, 4 * 64, dtype=dtype)
    angle = torch.rand(50, rot // 2, generator=g, device="cuda") * 6.28
    table = torch.cat([angle.cos(), angle.sin()], 1)
    clean = q.clone()
    x = q.view(9, 4, 64)
    x[1, 0, rot], x[2, 1, rot + 3], x[3, 2, 63], x[4, 3, rot + 6] = float("inf"), float("-inf"), float("nan"), float("inf")
    spoilt, pos = q.clone(), torch.arange(9, device="cuda")
    for t in (q, clean):
        capi.qk_norm_rotary_embedding(pos, t, None, 64, table, neox, eps=None)
    tail = torch.cat([t.view(9, 4, 64)[..., rot:].flatten().nan_to_num(7, 8, 9) for t in (q, spoilt)])
    assert torch.equal(tail[:tail.numel() // 2], tail[tail.numel() // 2:])
    assert torch.equal(q.view(9, 4, 64)[..., :rot], clean.view(9, 4, 64)[..., :rot])


@pytest.mark.parametrize("new,page", KERNELS)
def test_huge_keys_and_tiny_queries(cuda, new, page):
    """Keys of about 2^118 and queries of about 2^-118: ordinary scores."""
    b = Batch(91, [300, 700], [new, new], 8, 2, 128, page, torch.bfloat16, True)
    for i, n in enumerate(b.lengths):
        page_, place = places(b, i, range(n))
        b.ke[page_, place] += 118
    b.q = (b.q.float() * 2.0 ** -118).bfloat16()
    check(b, b.call())


@pytest.mark.parametrize("lengths,new,heads,kv_heads", [([3000], [60], 8, 2), ([5000, 300, 900], [1, 1, 1], 8, 2), ([700], [1], 32, 32), ([9000, 20], [4, 2], 8, 2)],
                         ids=["cluster", "line", "single", "few"])
@pytest.mark.parametrize("ahead", [0, 30])
def test_value_heads_of_zeros_where_several_ctas_share_a_sequence(cuda, lengths, new, heads, kv_heads, ahead):
    """Long runs of zero heads, so that some of the pieces that are joined have nothing else."""
    b = Batch(89, lengths, new, heads, kv_heads, 128, 16, torch.bfloat16, True)
    b.q[..., 0] = 4
    for i, n in enumerate(lengths):
        page, place = places(b, i, range(n))
        b.kc.view(torch.uint8)[page, place, :, 0] = 0
        b.ve[page, place] = (b.ve[page, place].int() - 20).to(torch.uint8)
        page, place = places(b, i, range(n // 8, n - n // 8))
        b.kc[page, place, :, 0] = torch.tensor(ahead * 128 ** 0.5 / 4 / 16, device="cuda").to(torch.float8_e4m3fn)
        b.vc.view(torch.uint8)[page, place] = 0
        b.ve[page, place] = 127
    for starts in (b.starts, None) if sum(new) == len(new) else (b.starts,):
        b.starts = starts
        check(b, b.call())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,new", [([300, 170], [40, 130]), ([4000, 70, 30], [2, 1, 1])], ids=["chunks", "few"])
def test_a_replayed_graph_of_a_batch_that_shrinks(cuda, e4m3, lengths, new):
    """A graph of fixed size: sequences that leave are padding in the next replay, and their rows are zeros."""
    b = Batch(92, lengths, new, 8, 2, 128, 16, torch.float16, e4m3)
    graph = torch.cuda.CUDAGraph()
    b.call()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = b.call()
    graph.replay()
    b.check(out)
    b.starts[-1] = b.starts[-2]
    want = b.call()
    graph.replay()
    torch.cuda.synchronize()
    live = sum(new[:-1])
    assert torch.equal(out, want) and bool((out[live:] == 0).all())
    b.starts.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((out == 0).all())
