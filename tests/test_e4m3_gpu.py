"""The paged cache of 8 bits on the GPU: storing keys and values, and attention over it, against 64 bits.

Bounds. A rounding to bfloat16 is off by 2^-8 of the value at most, one to e4m3 by 2^-4 (2^-10 scales below its normal range).
Attention rounds the weights (2^-8 of sum p |v|) and the output (2^-8); payloads, scales and their products in bfloat16 are exact; scores are float32
sums of d products: off by d 2^-23 of sum |q||k| scale, which moves a weight, and the sum of the weights, by as much; the special-function unit's
exponential adds 2^-21. Where weights are taken together with their values' scales, in float16 with 2^15 for the largest, those below 2^-14 are multiples
of 2^-24, so off by 2^-25, which is 2^-40 of the largest p_j scale_j, for every |v_j| / scale_j: what counts where the heaviest key's value is near zero and
others' scales are far from its own."""
import math

import pytest
import torch

import plain_e4m3 as plain
from vosti_b200 import ops

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def tables(limit, rotary):
    angle = torch.arange(limit, dtype=torch.float64).view(-1, 1) * 10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))
    return angle.cos().float(), angle.sin().float()


def store(cache, ctx, group, qkv, *, nq, nkv, d, norm=True, rotary=None, neighbours=False, gen=None, partial=None):
    """Runs the kernel over qkv (CPU) and compares queries, payloads and scales with 64 bits. Returns the cache's numbers before and after."""
    rotary = d if rotary is None else rotary
    w = [torch.randn(d, generator=gen) * 0.1 + 1 for _ in range(2)] if norm else [None, None]
    cos, sin = tables(int(ctx.positions.max()) + 3, rotary) if rotary else (None, None)
    cuda = lambda t: None if t is None else t.to(DEVICE)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    source = cuda(qkv)
    if partial:
        pieces = torch.randn(partial, *qkv.shape, generator=gen)
        pieces[-1] = qkv.float() - pieces[:-1].sum(0)
        source = ops.PartialSum(cuda(pieces).contiguous(), partial, *qkv.shape, torch.bfloat16, ctx.status)
        qkv = pieces.double().sum(0)
    q = ops.qkv_post_e4m3(source, cache, nq=nq, nkv=nkv, head_dim=d, q_norm_w=cuda(w[0]), k_norm_w=cuda(w[1]), eps=1e-6, cos=cuda(cos), sin=cuda(sin),
                          positions=ctx.positions, slot_mapping=group.slot_mapping, status=ctx.status, rotary_dim=rotary or d, interleaved=neighbours)
    assert int(ctx.status) == 0
    rows, pos = qkv.view(-1, nq + 2 * nkv, d), ctx.positions.cpu().long()
    after = lambda x, weight: plain.heads_after(x, weight, 1e-6, cos, sin, pos, rotary, neighbours)
    want_q = after(rows[:, :nq], w[0])
    size = want_q.abs().amax(-1, keepdim=True)
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -24
    assert bool(((q.cpu().double().view(want_q.shape) - want_q).abs() <= half * want_q.abs() + 3e-6 * size).all())
    page, blocks_a_page = cache.page_size, cache.page_size // 16
    slots = group.slot_mapping.cpu().tolist()
    runs = {}
    for t, s in enumerate(slots):
        if s >= 0:
            runs.setdefault(s // 16, []).append((t, s % 16))
    for name, want, old_payload, old_scale, payload, scale in (
            ("k", after(rows[:, nq:nq + nkv], w[1]), before[0], before[2], cache.k, cache.k_scale),
            ("v", rows[:, nq + nkv:].double(), before[1], before[3], cache.v, cache.v_scale)):
        by_block = lambda t: (t.cpu().view(torch.uint8).view(-1, nkv, blocks_a_page, d, 16) if name == "v"
                              else t.cpu().view(torch.uint8).view(-1, nkv, blocks_a_page, 16, d).transpose(-1, -2)).contiguous()
        old, new = by_block(old_payload), by_block(payload)
        old_s, new_s = old_scale.cpu().view(torch.uint8), scale.cpu().view(torch.uint8)
        expected, expected_s = old.clone(), old_s.clone()
        for block, tokens in runs.items():
            p, b, first = block // blocks_a_page, block % blocks_a_page, tokens[0][1]
            for g in range(nkv):
                fresh = torch.stack([want[t, g] for t, _ in tokens], dim=-1)                   # [d, n]
                need = plain.scale_for(float(fresh.abs().max()))
                byte = max(need, int(old_s[p, g, b])) if first else need
                got = int(new_s[p, g, b])
                assert got == byte, (name, block, g, got, byte)
                expected_s[p, g, b] = byte
                s = 2.0 ** (byte - 127)
                numbers = plain.held(new[p, g, b]) * s
                for i, (t, o) in enumerate(tokens):
                    x = fresh[:, i]
                    bound = torch.maximum(x.abs() * 2.0 ** -4, torch.tensor(s * 2.0 ** -10)) + 3e-6 * x.abs().max()
                    assert bool(((numbers[:, o] - x).abs() <= bound).all()), (name, block, g, t)
                    expected[p, g, b, :, o] = new[p, g, b, :, o]
                if first:
                    ratio = 2.0 ** (int(old_s[p, g, b]) - byte)
                    again = (plain.held(old[p, g, b][:, :first]) * ratio).float().to(torch.float8_e4m3fn).view(torch.uint8)
                    expected[p, g, b, :, :first] = again
        # all the rest, earlier tokens under their block's scale included, to the bit
        assert torch.equal(new_s, expected_s)
        zero = lambda t: torch.where(t == 128, 0, t)                                           # (-0 and 0 are one number)
        assert torch.equal(zero(new), zero(expected)), name
    return q


@pytest.mark.parametrize("new,past", [([1], [0]), ([1], [15]), ([1], [16]), ([1] * 9, [0, 1, 7, 15, 16, 17, 31, 32, 200]), ([16], [0]), ([17], [15]), ([5], [3]),
                                      ([33, 1, 2, 70], [5, 14, 15, 0]), ([130], [0]), ([64, 66], [1, 47]), ([3, 3, 3], [13, 14, 15])])
@pytest.mark.parametrize("dtype,nq,nkv,d,page", [(torch.bfloat16, 8, 2, 128, 16), (torch.float32, 4, 4, 64, 32), (torch.bfloat16, 3, 1, 80, 48),
                                                 (torch.bfloat16, 17, 1, 256, 16), (torch.bfloat16, 2, 1, 16, 16)])
def test_store(new, past, dtype, nq, nkv, d, page):
    gen = torch.Generator().manual_seed(sum(new) + d)
    ctx, group, pages = plain.step(new, past, page)
    cache = plain.random_cache(pages, nkv, page, d, gen, low=114, high=124)                     # scales above and below what the step needs
    store(cache, ctx, group, torch.randn(sum(new), (nq + 2 * nkv) * d, generator=gen).to(dtype), nq=nq, nkv=nkv, d=d, gen=gen)


@pytest.mark.parametrize("rotary,neighbours,norm", [(64, True, True), (32, False, True), (32, True, False), (0, False, True), (0, False, False), (64, False, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_rotations(rotary, neighbours, norm, dtype):
    gen = torch.Generator().manual_seed(5)
    ctx, group, pages = plain.step([21, 1, 1, 40], [9, 33, 0, 15], 16)
    cache = plain.random_cache(pages, 2, 16, 64, gen, low=114, high=124)
    store(cache, ctx, group, torch.randn(63, 8 * 64, generator=gen).to(dtype), nq=4, nkv=2, d=64, gen=gen, rotary=rotary, neighbours=neighbours, norm=norm)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 15, 16])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 256), (torch.bfloat16, 80), (torch.float32, 16)])
def test_store_of_a_norm_without_an_eps(n, dtype, d):
    """A run's lanes without a token hold zeros, whose norm is no number at eps 0: they do not count. A token of zeros does."""
    gen = torch.Generator().manual_seed(n + d)
    ctx, group, pages = plain.step([n], [0], 16)
    qkv = torch.randn(n, 4 * d, generator=gen).to(dtype)
    caches = [plain.random_cache(pages, 1, 16, d, torch.Generator().manual_seed(3)) for _ in range(2)]
    common = dict(nq=2, nkv=1, head_dim=d, k_norm_w=torch.ones(d, device=DEVICE), slot_mapping=group.slot_mapping, status=ctx.status)
    for cache, eps in zip(caches, (0.0, 1e-12)):                          # (1e-12 beside a mean square near 1 is nothing in float32)
        ops.qkv_post_e4m3(qkv.to(DEVICE), cache, eps=eps, **common)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8)), name
    at = int(group.block_table[0, 0])
    assert int(caches[0].k_scale.view(torch.uint8)[at, 0, 0]) != 255
    qkv[-1, 2 * d:3 * d] = 0
    ops.qkv_post_e4m3(qkv.to(DEVICE), caches[0], eps=0.0, **common)
    assert int(caches[0].k_scale.view(torch.uint8)[at, 0, 0]) == 255 and int(ctx.status) == 0


@pytest.mark.parametrize("splits", [1, 3, 7])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_store_of_unsummed_products(splits, d):
    gen = torch.Generator().manual_seed(splits)
    ctx, group, pages = plain.step([1] * 5, [0, 15, 40, 7, 100], 16)
    cache = plain.random_cache(pages, 2, 16, d, gen, low=114, high=124)
    store(cache, ctx, group, torch.randn(5, 8 * d, generator=gen), nq=4, nkv=2, d=d, gen=gen, partial=splits)


@pytest.mark.parametrize("size", [0.0, 1e-42, 1e-30, 448.0, 448.5, 3e4, 7.9e28, 1e30, 3e38])
def test_store_of_extreme_sizes(size):
    """From 2^96 on a size counts as no number: the attention's sums would pass float32."""
    gen = torch.Generator().manual_seed(7)
    ctx, group, pages = plain.step([20], [0], 16)
    cache = plain.random_cache(pages, 1, 16, 64, gen)
    qkv = torch.rand(20, 3 * 64, generator=gen) * 2 - 1
    qkv[:, ::7] = 1.0
    if size >= 2.0 ** 96:
        ops.qkv_post_e4m3((qkv * size).to(DEVICE), cache, nq=1, nkv=1, head_dim=64, slot_mapping=group.slot_mapping, status=ctx.status)
        at = group.block_table[0, :2].long()
        assert bool((cache.k_scale.view(torch.uint8)[at] == 255).all()) and bool((cache.v_scale.view(torch.uint8)[at] == 255).all())
        return
    store(cache, ctx, group, qkv * size, nq=1, nkv=1, d=64, gen=gen, rotary=0, norm=False)


def test_store_from_one_word_on():
    """A projection that does not start on whole words."""
    gen = torch.Generator().manual_seed(9)
    ctx, group, pages = plain.step([9], [4], 16)
    qkv = torch.randn(9, 4 * 128, generator=gen).bfloat16()
    odd = torch.zeros(9 * 512 + 1, dtype=torch.bfloat16, device=DEVICE)[1:].view(9, 512)
    odd.copy_(qkv)
    caches = [plain.random_cache(pages, 1, 16, 128, torch.Generator().manual_seed(3)) for _ in range(2)]
    cos, sin = (t.to(DEVICE) for t in tables(64, 128))
    common = dict(nq=2, nkv=1, head_dim=128, cos=cos, sin=sin, positions=ctx.positions, slot_mapping=group.slot_mapping, status=ctx.status)
    a, b = ops.qkv_post_e4m3(qkv.to(DEVICE), caches[0], **common), ops.qkv_post_e4m3(odd, caches[1], **common)
    assert torch.equal(a, b)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8))


def test_tokens_without_a_slot_and_faults():
    gen = torch.Generator().manual_seed(11)
    ctx, group, pages = plain.step([20], [0], 16)
    cache = plain.random_cache(pages, 1, 16, 64, gen)
    before = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    qkv = torch.randn(20, 3 * 64, generator=gen).to(DEVICE)
    common = dict(nq=1, nkv=1, head_dim=64, status=ctx.status)

    def unchanged():
        return all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    ops.qkv_post_e4m3(qkv, cache, slot_mapping=torch.full((20,), -1, dtype=torch.int32, device=DEVICE), **common)
    assert unchanged() and int(ctx.status) == 0
    for bad in (pages * 16, -2, 2 ** 31 - 1):
        ops.qkv_post_e4m3(qkv, cache, slot_mapping=torch.full((20,), bad, dtype=torch.int32, device=DEVICE), **common)
        assert unchanged() and int(ctx.status) == 2
        ctx.status.zero_()
    # one slot twice, and a block's tokens out of order: reported, and only the first of them is stored
    for slots in ([3, 3], [3, 2]):
        ops.qkv_post_e4m3(qkv[:2], cache, slot_mapping=torch.tensor(slots, dtype=torch.int32, device=DEVICE), **common)
        assert int(ctx.status) == 2
        ctx.status.zero_()
    # a position beyond the tables
    cos, sin = (t.to(DEVICE) for t in tables(4, 64))
    ops.qkv_post_e4m3(qkv, cache, slot_mapping=group.slot_mapping, cos=cos, sin=sin, positions=ctx.positions, **common)
    assert int(ctx.status) == 8


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_value_that_is_not_finite_marks_its_block(bad):
    gen = torch.Generator().manual_seed(13)
    ctx, group, pages = plain.step([40], [0], 16, shuffled=False)
    cache = ops.PagedE4M3.zeros(pages, 2, 16, 64)
    qkv = torch.randn(40, 5 * 64, generator=gen)
    qkv[18, 64 * 1 + 5] = bad                         # key of head 0, block 1
    qkv[33, 64 * 4 + 9] = bad                         # value of head 1, block 2
    ops.qkv_post_e4m3(qkv.to(DEVICE), cache, nq=1, nkv=2, head_dim=64, slot_mapping=group.slot_mapping, status=ctx.status)
    keys, values = plain.dequantized(cache)
    assert keys[1, 0].isnan().all() and keys.isnan().sum() == 16 * 64
    assert values[2, 1].isnan().all() and values.isnan().sum() == 16 * 64
    a, b = cache.dequantized()
    assert torch.equal(a.cpu().double().nan_to_num(7.0), keys.nan_to_num(7.0)) and torch.equal(b.cpu().double().nan_to_num(7.0), values.nan_to_num(7.0))
    # the next tenant of the page starts afresh
    ctx, group, _ = plain.step([20], [0], 16, shuffled=False)
    ops.qkv_post_e4m3(torch.randn(20, 5 * 64, generator=gen).to(DEVICE), cache, nq=1, nkv=2, head_dim=64, slot_mapping=group.slot_mapping, status=ctx.status)
    keys, _ = plain.dequantized(cache)
    assert not keys[0].isnan().any() and not keys[1, :, :4].isnan().any()


# ---------------------------------------------------------------- attention
def check_attention(q, cache, ctx, group, out, *, nq, nkv, d, window, scale):
    keys, values = plain.dequantized(cache)
    v_scales = plain.scales(cache.v_scale).repeat_interleave(16, dim=2)
    at = 0
    for r, (n, total) in enumerate(zip(ctx.host_q_lens, ctx.host_kv_lens)):
        page, place = plain.rows_of(group.block_table[r], total, group.page_size)
        k, v = keys[page, :, place].transpose(0, 1), values[page, :, place].transpose(0, 1)
        s = v_scales[page, :, place].transpose(0, 1)
        want, spread, reach, beside = plain.attend(q[at:at + n].cpu().view(n, nq, d), k, v, pos=torch.arange(total - n, total), nq=nq, nkv=nkv, scale=scale, window=window,
                                                   value_scales=s)
        got = out[at:at + n].cpu().double().view(n, nq, d)
        half = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -22
        bound = half * (spread + want.abs()) + 2 * (d * 2.0 ** -23 * reach + 2.0 ** -21) * spread + total * 2.0 ** -24 * spread + 2.0 ** -40 * beside
        assert torch.equal(got.isnan(), want.isnan())
        worst = ((got - want).abs() - bound).nan_to_num(0.0).max()
        assert float(worst) <= 0, (r, float(worst))
        at += n


def attention(new, past, *, nq, nkv, d, page=16, window=0, dtype=torch.bfloat16, seed=0, sharp=1.0, poison=True, low=117, high=123):
    gen = torch.Generator().manual_seed(seed + 3)
    ctx, group, pages = plain.step(new, past, page, seed=seed)
    cache = plain.random_cache(pages, nkv, page, d, gen, low=low, high=high)
    if poison:
        # slots that no token holds, and pages that no request holds: payloads that are no numbers
        used = torch.zeros(pages, page, dtype=torch.bool)
        for r, total in enumerate(ctx.host_kv_lens):
            used[plain.rows_of(group.block_table[r], total, page)] = True
        free = ~used
        k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
        k.masked_fill_(free.to(DEVICE).view(pages, 1, page, 1), 127)
        v.masked_fill_(free.to(DEVICE).view(pages, 1, page // 16, 1, 16), 127)
        whole = free.view(pages, page // 16, 16).all(-1).view(pages, 1, page // 16).to(DEVICE)
        cache.k_scale.view(torch.uint8).masked_fill_(whole, 255)
        cache.v_scale.view(torch.uint8).masked_fill_(whole, 255)
    q = (torch.randn(sum(new), nq * d, generator=gen) * sharp).to(dtype).to(DEVICE)
    scale = d ** -0.5
    out = ops.attention_e4m3(ctx, q, cache, group, nq=nq, nkv=nkv, head_dim=d, scale=scale, window=window)
    assert int(ctx.status) == 0
    check_attention(q, cache, ctx, group, out, nq=nq, nkv=nkv, d=d, window=window, scale=scale)
    return q, cache, ctx, group, out


LENGTHS = [([1], [0]), ([1], [1]), ([1], [14]), ([1], [15]), ([1], [16]), ([1], [63]), ([1], [64]), ([1], [700]), ([1] * 5, [0, 17, 255, 256, 1500]),
           ([1] * 40, [(i * 97) % 800 for i in range(40)]), ([2, 4, 1], [30, 0, 100])]


@pytest.mark.parametrize("new,past", LENGTHS)
@pytest.mark.parametrize("nq,nkv,d,page", [(32, 8, 128, 16), (4, 4, 64, 32), (5, 1, 128, 48), (16, 1, 64, 16), (40, 2, 128, 64)])
def test_single_tokens(new, past, nq, nkv, d, page):
    attention(new, past, nq=nq, nkv=nkv, d=d, page=page, seed=len(new))


@pytest.mark.parametrize("window", [1, 2, 16, 17, 64, 100, 5000])
@pytest.mark.parametrize("new,past", [([1] * 4, [0, 20, 150, 900]), ([70, 9], [130, 40]), ([300], [0])])
def test_windows(window, new, past):
    attention(new, past, nq=8, nkv=2, d=128, window=window)
    attention(new, past, nq=3, nkv=1, d=64, page=32, window=window)


@pytest.mark.parametrize("new,past", [([5], [0]), ([16], [0]), ([17], [15]), ([63], [1]), ([64], [64]), ([65], [0]), ([129], [500]), ([300, 7, 1, 1], [0, 90, 33, 4]),
                                      ([40, 6, 2, 3], [77, 0, 200, 31]), ([513], [0])])
@pytest.mark.parametrize("nq,nkv,d,page", [(32, 8, 128, 16), (6, 2, 64, 32), (5, 1, 128, 48), (16, 1, 128, 16), (20, 1, 64, 16)])
def test_portions(new, past, nq, nkv, d, page):
    attention(new, past, nq=nq, nkv=nkv, d=d, page=page, seed=3)


@pytest.mark.parametrize("new,past", [([300], [1200]), ([20], [1500]), ([5], [3000]), ([130, 7, 1], [900, 2000, 50]), ([64], [700]), ([512], [600])])
@pytest.mark.parametrize("nq,nkv,d,page,window", [(32, 8, 128, 16, 0), (6, 2, 64, 32, 0), (16, 1, 128, 16, 0), (8, 8, 64, 64, 900), (5, 1, 128, 48, 600)])
def test_portions_behind_long_caches(new, past, nq, nkv, d, page, window):
    """Few rows, many keys: the keys are cut over CTAs."""
    attention(new, past, nq=nq, nkv=nkv, d=d, page=page, window=window, seed=4)


@pytest.mark.parametrize("d", [64, 128])
def test_a_long_cache_beside_a_portion_does_not_cut_its_keys(d):
    """How a portion's keys are cut goes by the portions of a step: the same bits beside a single token that sees many more."""
    gen = torch.Generator().manual_seed(6)
    ctx, group, pages = plain.step([300, 1], [0, 3500], 16)
    cache = plain.random_cache(pages, 1, 16, d, gen)
    q = torch.randn(301, 4 * d, generator=gen).bfloat16().to(DEVICE)
    sizes = dict(nq=4, nkv=1, head_dim=d, scale=d ** -0.5)
    both = ops.attention_e4m3(ctx, q, cache, group, **sizes)
    check_attention(q, cache, ctx, group, both, nq=4, nkv=1, d=d, window=0, scale=d ** -0.5)
    alone, view, _ = plain.step([300], [0], 16)
    view.block_table = group.block_table[:1]
    assert torch.equal(ops.attention_e4m3(alone, q[:300], cache, view, **sizes), both[:300]) and int(ctx.status) == int(alone.status) == 0


def test_segments_of_both_head_sizes():
    """One token of few heads behind many keys, for each head size first or after the other."""
    for d in (64, 128, 64):
        attention([1], [9000], nq=2, nkv=1, d=d, page=64)


@pytest.mark.parametrize("side", ["k_scale", "v_scale"])
def test_segments_that_are_no_number(side):
    gen = torch.Generator().manual_seed(4)
    ctx, group, pages = plain.step([40, 1], [1000, 600], 16)
    cache = plain.random_cache(pages, 1, 16, 128, gen)
    first, middle = (int(group.block_table[0, i]) for i in (0, 40))
    for blocks in ([middle], [first, middle], [int(p) for p in group.block_table[0, :16]]):
        for b in blocks:
            getattr(cache, side).view(torch.uint8)[b, 0, 0] = 255
        for window in (0, 100):
            q = torch.randn(41, 2 * 128, generator=gen).bfloat16().to(DEVICE)
            out = ops.attention_e4m3(ctx, q, cache, group, nq=2, nkv=1, head_dim=128, scale=0.09, window=window)
            check_attention(q, cache, ctx, group, out, nq=2, nkv=1, d=128, window=window, scale=0.09)


@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1], [40, 300]), ([70, 1, 5], [30, 64, 0])])
@pytest.mark.parametrize("dtype,nq,nkv,d,window", [(torch.float32, 4, 2, 128, 0), (torch.float32, 3, 3, 80, 33), (torch.bfloat16, 4, 1, 96, 0), (torch.bfloat16, 2, 2, 256, 40),
                                                   (torch.float32, 2, 1, 16, 0)])
def test_on_the_cuda_cores(new, past, dtype, nq, nkv, d, window):
    attention(new, past, nq=nq, nkv=nkv, d=d, dtype=dtype, window=window)


@pytest.mark.parametrize("new,past", [([1], [900]), ([100], [200])])
@pytest.mark.parametrize("sharp,low,high", [(20.0, 117, 123), (1e-3, 0, 3), (1e-3, 60, 140), (1.0, 100, 110)])
def test_extreme_scores_and_scales(new, past, sharp, low, high):
    """Weights of one key alone, scales near the smallest and far apart."""
    attention(new, past, nq=4, nkv=1, d=64, sharp=sharp, low=low, high=high)
    attention(new, past, nq=4, nkv=1, d=64, sharp=sharp, low=low, high=high, dtype=torch.float32)


@pytest.mark.parametrize("exponent", [134, 135, 140, 200, 215])
def test_scales_above_one_factor(exponent):
    """Scales whose payload bits need two factors to become bfloat16, up to the largest that sizes below 2^96 are given
    (2^96 = 256 * 2^88; with 448 * 2^119 the sum of two keys' values passes float32 before it is divided)."""
    for new, past in (([1], [100]), ([40], [30])):
        gen = torch.Generator().manual_seed(2)
        ctx, group, pages = plain.step(new, past, 16)
        cache = plain.random_cache(pages, 1, 16, 64, gen, low=120, high=121)
        cache.v_scale.view(torch.uint8).fill_(exponent)
        q = torch.randn(sum(new), 64, generator=gen).bfloat16().to(DEVICE)
        out = ops.attention_e4m3(ctx, q, cache, group, nq=1, nkv=1, head_dim=64, scale=0.125)
        check_attention(q, cache, ctx, group, out, nq=1, nkv=1, d=64, window=0, scale=0.125)


@pytest.mark.parametrize("new,past", [([1] * 6, [10, 17, 31, 32, 40, 200]), ([60], [0]), ([50, 1], [20, 40])])
@pytest.mark.parametrize("side", ["k_scale", "v_scale"])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
def test_a_block_that_is_no_number_reaches_only_who_sees_it(new, past, side, d, dtype):
    gen = torch.Generator().manual_seed(4)
    ctx, group, pages = plain.step(new, past, 16)
    cache = plain.random_cache(pages, 1, 16, d, gen)
    for r, total in enumerate(ctx.host_kv_lens):
        if total > 32:
            getattr(cache, side).view(torch.uint8)[int(group.block_table[r, 2]), 0, 0] = 255     # keys 32 .. 47
    for window in (0, 8):
        q = torch.randn(sum(new), 2 * d, generator=gen).to(dtype).to(DEVICE)
        out = ops.attention_e4m3(ctx, q, cache, group, nq=2, nkv=1, head_dim=d, scale=d ** -0.5, window=window)
        assert out.isnan().any()
        check_attention(q, cache, ctx, group, out, nq=2, nkv=1, d=d, window=window, scale=d ** -0.5)


@pytest.mark.parametrize("new,past", [([1] * 4, [10, 33, 40, 200]), ([60], [0]), ([50, 1], [20, 40]), ([70], [1400])])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("byte", [0x7f, 0xff])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
def test_a_payload_that_is_no_number_reaches_only_who_sees_it(new, past, side, byte, d, dtype):
    """One of a key makes the rows that see it no numbers, one of a value their feature at least; the same for single tokens, portions and the CUDA cores."""
    gen = torch.Generator().manual_seed(5)
    ctx, group, pages = plain.step(new, past, 16)
    cache = plain.random_cache(pages, 1, 16, d, gen)
    for r, total in enumerate(ctx.host_kv_lens):
        for token, feature in ((33, 7), (45, d - 1)):
            if total > token:
                page, place = int(group.block_table[r, token // 16]), token % 16
                at = (page, 0, place, feature) if side == "k" else (page, 0, 0, feature, place)
                getattr(cache, side).view(torch.uint8)[at] = byte
    for window in (0, 5, 8):
        q = torch.randn(sum(new), 2 * d, generator=gen).to(dtype).to(DEVICE)
        out = ops.attention_e4m3(ctx, q, cache, group, nq=2, nkv=1, head_dim=d, scale=d ** -0.5, window=window)
        heads = out.view(-1, 2, d)
        if side == "v":                                   # the rest of such a row is a number or none
            heads = torch.where(heads[..., [7, d - 1]].isnan().any(-1, keepdim=True), torch.nan, heads)
        check_attention(q, cache, ctx, group, heads.reshape(out.shape), nq=2, nkv=1, d=d, window=window, scale=d ** -0.5)


def test_pages_beyond_the_pool_are_reported():
    gen = torch.Generator().manual_seed(6)
    for new, past, dtype in (([1], [100], torch.bfloat16), ([40], [60], torch.bfloat16), ([1], [100], torch.float32)):
        ctx, group, pages = plain.step(new, past, 16)
        cache = plain.random_cache(pages, 1, 16, 64, gen)
        q = torch.randn(sum(new), 64, generator=gen).to(dtype).to(DEVICE)
        for bad in (pages, -1):
            group.block_table[0, 1] = bad
            ops.attention_e4m3(ctx, q, cache, group, nq=1, nkv=1, head_dim=64, scale=0.125)
            assert int(ctx.status) == 4
            ctx.status.zero_()


def test_long_cache():
    """More than 2^31 bytes of keys: offsets pass 32 bits. One request at the pool's end."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 12 GB")
    heads, page, d = 8, 64, 128
    pages = (1 << 31) // (heads * page * d) * 2 + 40
    cache = ops.PagedE4M3.zeros(pages, heads, page, d)
    gen = torch.Generator().manual_seed(8)
    for new, past in (([1], [500]), ([130], [200])):
        ctx, group, need = plain.step(new, past, page, shuffled=False)
        group.block_table.add_(torch.where(group.block_table >= 0, pages - need, 0))
        group.slot_mapping.add_((pages - need) * page)
        small = plain.random_cache(need, heads, page, d, gen)
        for name in ("k", "v", "k_scale", "v_scale"):
            getattr(cache, name).view(torch.uint8)[-need:] = getattr(small, name).view(torch.uint8)
        qkv = torch.randn(sum(new), 24 * d, generator=gen).bfloat16().to(DEVICE)
        q = ops.qkv_post_e4m3(qkv, cache, nq=8, nkv=8, head_dim=d, slot_mapping=group.slot_mapping, status=ctx.status)
        out = ops.attention_e4m3(ctx, q, cache, group, nq=8, nkv=8, head_dim=d, scale=d ** -0.5)
        assert int(ctx.status) == 0
        tail = ops.PagedE4M3(*(getattr(cache, name)[-need:].clone() for name in ("k", "v", "k_scale", "v_scale")))
        group.block_table.sub_(torch.where(group.block_table >= 0, pages - need, 0))
        check_attention(q, tail, ctx, group, out, nq=8, nkv=8, d=d, window=0, scale=d ** -0.5)
        assert int(cache.k.view(torch.uint8)[:-need].count_nonzero()) == 0 if past == [500] else True


def test_another_stream_and_a_graph():
    """On a stream of its own and replayed from a recording the answers are the same bits."""
    gen = torch.Generator().manual_seed(15)
    ctx, group, pages = plain.step([1] * 3, [40, 700, 15], 16)
    caches = [plain.random_cache(pages, 2, 16, 128, torch.Generator().manual_seed(1)) for _ in range(3)]
    qkv = torch.randn(3, 8 * 128, generator=gen).bfloat16().to(DEVICE)

    def run(cache):
        q = ops.qkv_post_e4m3(qkv, cache, nq=4, nkv=2, head_dim=128, slot_mapping=group.slot_mapping, status=ctx.status)
        return ops.attention_e4m3(ctx, q, cache, group, nq=4, nkv=2, head_dim=128, scale=0.09)
    want = run(caches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    run(caches[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run(caches[2])
    for _ in range(2):
        kept.zero_()
        graph.replay()
        assert torch.equal(kept, want)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("new,past", [([1], [0]), ([1] * 3, [15, 16, 700]), ([1] * 9, [0, 63, 64, 65, 127, 128, 1000, 2047, 31]), ([4, 1, 3], [60, 61, 190]), ([70, 1, 4, 1], [30, 500, 126, 64]),
                                      ([1] * 70, [(i * 131) % 900 for i in range(70)])])
@pytest.mark.parametrize("nq,nkv,d,window", [(32, 8, 128, 0), (4, 2, 64, 0), (8, 1, 128, 40), (24, 1, 64, 0)])
def test_attention_right_behind_the_store(new, past, nq, nkv, d, window):
    """What is read while the store still runs is what stands there after it: with blocks whose scale grows, so that their earlier tokens
    are rounded again, the same bits as from a call that waits."""
    gen = torch.Generator().manual_seed(len(new) + nq)
    ctx, group, pages = plain.step(new, past, 16, seed=7)
    first = [plain.random_cache(pages, nkv, 16, d, gen, low=100, high=120) for _ in range(4)]
    qkv = [(torch.randn(sum(new), (nq + 2 * nkv) * d, generator=gen) * 3).bfloat16().to(DEVICE) for _ in first]
    copies = lambda: [ops.PagedE4M3(*(getattr(c, n).view(torch.uint8).clone().view(getattr(c, n).dtype) for n in ("k", "v", "k_scale", "v_scale"))) for c in first]
    sizes = dict(nq=nq, nkv=nkv, head_dim=d)

    def run(caches, outs, **more):
        for cache, x in zip(caches, qkv):
            q = ops.qkv_post_e4m3(x, cache, slot_mapping=group.slot_mapping, status=ctx.status, **sizes)
            outs.append(ops.attention_e4m3(ctx, q, cache, group, scale=d ** -0.5, window=window, **sizes, **more))
            if not more:
                torch.cuda.synchronize()
    slow, fast = copies(), copies()
    want, got = [], []
    run(slow, want)
    run(fast, got, appended=ctx.max_q_len)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(fast, slow):
        assert all(torch.equal(getattr(a, n).view(torch.uint8), getattr(b, n).view(torch.uint8)) for n in ("k", "v", "k_scale", "v_scale"))
    check_attention(ops.qkv_post_e4m3(qkv[0], copies()[0], slot_mapping=group.slot_mapping, status=ctx.status, **sizes), fast[0], ctx, group, got[0], nq=nq, nkv=nkv, d=d,
                    window=window, scale=d ** -0.5)
    again, kept = copies(), []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(again, kept, appended=ctx.max_q_len)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(kept, want)) and int(ctx.status) == 0


@pytest.mark.parametrize("d,count", [(128, 1), (128, 40), (64, 3), (96, 2)])
def test_tokens_of_a_block_one_after_another(d, count):
    """Stores that follow one another without a pause, each with larger values than the last: every one of them rounds what the block holds again."""
    gen = torch.Generator().manual_seed(5)
    steps = [plain.step([1] * count, [p] * count, 16, seed=2, spare=2 if p > 15 else 2 + count) for p in range(12, 24)]
    ctx, group, pages = steps[-1]
    rows = [(torch.randn(count, 4 * d, generator=gen) * 1.7 ** i).bfloat16().to(DEVICE) for i in range(len(steps))]
    table = group.block_table.cpu()
    slots = [torch.tensor([int(table[r, p // 16]) * 16 + p % 16 for r in range(count)], dtype=torch.int32, device=DEVICE) for p in range(12, 24)]
    kept = []
    for wait in (True, False):
        cache = plain.random_cache(pages, 1, 16, d, torch.Generator().manual_seed(9), low=90, high=100)
        torch.cuda.synchronize()
        for x, slot in zip(rows, slots):
            ops.qkv_post_e4m3(x, cache, nq=2, nkv=1, head_dim=d, slot_mapping=slot, status=ctx.status)
            if wait:
                torch.cuda.synchronize()
        kept.append([getattr(cache, n).view(torch.uint8).clone() for n in ("k", "v", "k_scale", "v_scale")])
    assert all(torch.equal(a, b) for a, b in zip(*kept)) and int(ctx.status) == 0


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 96)])
def test_a_step_without_tokens(dtype, d):
    ctx, group, pages = plain.step([3], [20], 16)
    cache = plain.random_cache(pages, 2, 16, d, torch.Generator().manual_seed(1))
    before = [getattr(cache, n).view(torch.uint8).clone() for n in ("k", "v", "k_scale", "v_scale")]
    sizes = dict(nq=4, nkv=2, head_dim=d)
    none = torch.zeros(0, dtype=torch.int32, device=DEVICE)
    cos, sin = (t.to(DEVICE) for t in tables(8, d))
    q = ops.qkv_post_e4m3(torch.zeros(0, 8 * d, dtype=dtype, device=DEVICE), cache, slot_mapping=none, positions=none, cos=cos, sin=sin, status=ctx.status, **sizes)
    assert tuple(q.shape) == (0, 4 * d) and q.dtype == dtype
    ctx.positions = ctx.request_of = none
    ctx.layout = {"attention": ops.attention_step_layout([])[1]}
    for table in (group.block_table, group.block_table[:0]):
        group.block_table = table
        out = ops.attention_e4m3(ctx, q, cache, group, scale=0.1, **sizes)
        assert tuple(out.shape) == (0, 4 * d) and out.dtype == dtype
    assert all(torch.equal(a, getattr(cache, n).view(torch.uint8)) for a, n in zip(before, ("k", "v", "k_scale", "v_scale"))) and int(ctx.status) == 0


def test_calls_that_are_refused():
    ctx, group, pages = plain.step([2, 40], [5, 0], 16)
    cache = ops.PagedE4M3.zeros(pages, 2, 16, 64)
    x = torch.zeros(42, 8 * 64, dtype=torch.bfloat16, device=DEVICE)
    cos = torch.ones(64, 32, device=DEVICE)
    good = dict(nq=4, nkv=2, head_dim=64, slot_mapping=group.slot_mapping, status=ctx.status)
    ops.qkv_post_e4m3(x, cache, **good)
    w64, w32 = torch.ones(64, dtype=torch.bfloat16, device=DEVICE), torch.ones(32, dtype=torch.bfloat16, device=DEVICE)
    for bad, more in ((x[0], {}), (x.half(), {}), (x.cpu(), {}), (x[:, :-64], {}), (x.t().contiguous().t(), {}), (x, dict(nkv=4)), (x, dict(nq=0, nkv=4)), (x, dict(head_dim=128)),
                      (x, dict(slot_mapping=group.slot_mapping[:5])), (x, dict(slot_mapping=group.slot_mapping.long())), (x, dict(slot_mapping=group.slot_mapping.cpu())),
                      (x, dict(status=ctx.status.float())), (x, dict(cos=cos, sin=cos)), (x, dict(cos=cos, positions=ctx.positions)),
                      (x, dict(cos=cos, sin=cos[:, :16], positions=ctx.positions)), (x, dict(cos=cos.double(), sin=cos, positions=ctx.positions)),
                      (x, dict(cos=cos, sin=cos, positions=ctx.positions[:3])), (x, dict(cos=cos, sin=cos, positions=ctx.positions, rotary_dim=128)),
                      (x, dict(q_norm_w=w32)), (x, dict(k_norm_w=w64.float(), q_norm_w=w64))):
        with pytest.raises(ops.KernelError):
            ops.qkv_post_e4m3(bad, cache, **{**good, **more})
    q = torch.zeros(42, 4 * 64, dtype=torch.bfloat16, device=DEVICE)
    good = dict(nq=4, nkv=2, head_dim=64, scale=0.1)
    ops.attention_e4m3(ctx, q, cache, group, **good)
    for bad, more in ((q[0], {}), (q.half(), {}), (q.cpu(), {}), (q[:, :-64], {}), (q.t().contiguous().t(), {}), (q, dict(nkv=4)), (q, dict(nq=5)), (q, dict(nkv=0)),
                      (q, dict(head_dim=32)), (q, dict(scale=0.0)), (q, dict(scale=math.nan)), (q, dict(window=-1)), (q, dict(appended=-1))):
        with pytest.raises(ops.KernelError):
            ops.attention_e4m3(ctx, bad, cache, group, **{**good, **more})
    for owner, name, bad in ((ctx, "positions", ctx.positions[:7]), (ctx, "request_of", ctx.request_of.long()), (ctx, "cu_q", ctx.cu_q.long()), (ctx, "kv_len", ctx.kv_len.cpu()),
                             (ctx, "status", ctx.status.long()), (group, "block_table", group.block_table.long()), (group, "block_table", group.block_table[0]),
                             (group, "page_size", 32)):
        kept = getattr(owner, name)
        setattr(owner, name, bad)
        with pytest.raises(ops.KernelError):
            ops.attention_e4m3(ctx, q, cache, group, **good)
        setattr(owner, name, kept)
    assert int(ctx.status) == 0


def test_arrays_with_too_few_requests_are_refused():
    """Portions read where the request behind theirs begins; nothing is launched on shorter arrays."""
    for new in ([5, 40], [2, 40], [40, 2]):
        ctx, group, pages = plain.step(new, [5, 0], 16)
        cache = plain.random_cache(pages, 1, 16, 64, torch.Generator().manual_seed(1))
        q = torch.zeros(sum(new), 2 * 64, dtype=torch.bfloat16, device=DEVICE)
        sizes = dict(nq=2, nkv=1, head_dim=64, scale=0.1)
        ops.attention_e4m3(ctx, q, cache, group, **sizes)
        for owner, name, bad in ((ctx, "cu_q", ctx.cu_q[:-1]), (ctx, "kv_len", ctx.kv_len[:-1]), (group, "block_table", group.block_table[:-1]),
                                 (ctx, "layout", {"attention": {**ctx.layout["attention"], "num_long_rows": 3}}),
                                 (ctx, "layout", {"attention": {**ctx.layout["attention"], "num_short_tokens": sum(new) + 1}}), (ctx, "num_tokens", sum(new) + 1)):
            kept = getattr(owner, name)
            setattr(owner, name, bad)
            with pytest.raises(ops.KernelError):
                ops.attention_e4m3(ctx, q, cache, group, **sizes)
            setattr(owner, name, kept)
        assert int(ctx.status) == 0


def test_a_layout_that_takes_short_requests_for_portions():
    """Which requests are portions is the layout's to say, few tokens or many."""
    ctx, group, pages = plain.step([3, 1, 2], [20, 500, 70], 16)
    cache = plain.random_cache(pages, 2, 16, 64, torch.Generator().manual_seed(2))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    ctx.layout = {"attention": dict(num_short_tokens=1, num_long_rows=2, max_long_q_len=3)}
    ctx.extras = {"attention.short_tokens": ints(3), "attention.long_rows": ints(0, 2)}
    q = torch.randn(6, 8 * 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEVICE)
    out = ops.attention_e4m3(ctx, q, cache, group, nq=8, nkv=2, head_dim=64, scale=0.125)
    assert int(ctx.status) == 0
    check_attention(q, cache, ctx, group, out, nq=8, nkv=2, d=64, window=0, scale=0.125)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 96)])
@pytest.mark.parametrize("window", [0, 20])
def test_rows_that_see_nothing_are_zeros(dtype, d, window):
    """A single token at position -1 (a place of a batch that no request fills) reads no page and comes out as zeros."""
    ctx, group, pages = plain.step([1] * 5, [10, 300, 2000, 0, 64], 16)
    cache = plain.random_cache(pages, 2, 16, d, torch.Generator().manual_seed(2))
    q = torch.randn(5, 4 * d, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEVICE)
    sizes = dict(nq=4, nkv=2, head_dim=d, scale=0.1, window=window)
    want = ops.attention_e4m3(ctx, q, cache, group, **sizes)
    ctx.positions[1] = ctx.positions[4] = -1
    group.block_table[1] = group.block_table[4] = -1
    for appended in (0, 1):
        out = ops.attention_e4m3(ctx, q, cache, group, appended=appended, **sizes)
        assert torch.equal(out[[0, 2, 3]], want[[0, 2, 3]]) and int(out[[1, 4]].count_nonzero()) == 0 and int(ctx.status) == 0


def test_two_streams_at_once():
    """Calls on two streams share nothing: both give what each gives alone."""
    steps = [plain.step(new, past, 16, seed=i) for i, (new, past) in enumerate((([1] * 8, [900] * 8), ([200, 1, 1], [100, 700, 40])))]
    gens = [torch.Generator().manual_seed(20 + i) for i in range(2)]
    caches = [[plain.random_cache(pages, 2, 16, 128, torch.Generator().manual_seed(i)) for _ in range(2)] for i, (_, _, pages) in enumerate(steps)]
    qkv = [torch.randn(ctx.num_tokens, 12 * 128, generator=g).bfloat16().to(DEVICE) for (ctx, _, _), g in zip(steps, gens)]

    def run(i, cache, turns):
        ctx, group, _ = steps[i]
        for _ in range(turns):
            q = ops.qkv_post_e4m3(qkv[i], cache, nq=8, nkv=2, head_dim=128, slot_mapping=group.slot_mapping, status=ctx.status)
            out = ops.attention_e4m3(ctx, q, cache, group, nq=8, nkv=2, head_dim=128, scale=0.09, appended=ctx.max_q_len)
        return out
    want = [run(i, caches[i][0], 20) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            got[i] = run(i, caches[i][1], 20)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(int(ctx.status) == 0 for ctx, _, _ in steps)
