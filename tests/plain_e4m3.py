"""The cache of 8 bits and its attention in 64 bits, from their definition, on the CPU."""
import math
from types import SimpleNamespace

import torch

from vosti_b200 import ops

BLOCK = 16


def held(payload):
    """What float8_e4m3fn bytes stand for; 0x7f and 0xff are no numbers."""
    b = payload.cpu().view(torch.uint8).long()
    sign, e, m = b >> 7, (b >> 3) & 15, (b & 7).double()
    size = torch.where(e > 0, (8 + m) * 2.0 ** (e - 10).double(), m * 2.0 ** -9)
    return torch.where((b & 127) == 127, torch.nan, torch.where(sign == 1, -size, size))


def scales(scale):
    b = scale.cpu().view(torch.uint8).double()
    return torch.where(b == 255, torch.nan, 2.0 ** (b - 127))


def dequantized(cache):
    """Keys and values [pages, kv heads, page, d] that a cache stands for."""
    each = lambda s: scales(s).repeat_interleave(BLOCK, dim=2).unsqueeze(-1)
    return held(cache.k) * each(cache.k_scale), held(cache.v).transpose(-1, -2).reshape(cache.k.shape) * each(cache.v_scale)


def scale_for(most):
    """Byte of the smallest power of two that brings `most` to 448 or below."""
    if most == 0:
        return 0
    m, p = math.frexp(most)
    return max(0, p - 9 + (m > 0.875) + 127)


def heads_after(x, w, eps, cos, sin, pos, rotary, neighbours):
    """Norm and rotation of head rows [T, heads, d] in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    if cos is None:
        return x
    pairs = torch.arange(rotary // 2)
    a, b = (2 * pairs, 2 * pairs + 1) if neighbours else (pairs, pairs + rotary // 2)
    c, s = cos.double()[pos].unsqueeze(1), sin.double()[pos].unsqueeze(1)
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def attend(q, keys, values, *, pos, nq, nkv, scale, window, value_scales=None):
    """(out, spread, reach) of one request's query rows q [n, nq, d] at positions `pos` over keys and values [nkv, kv, d]: the
    output, sum_j p_j |v_j|, and the largest scale * sum |q||k| (what the error bounds are made of). With the values' scales [nkv, kv] also the
    largest p_j scale_j times sum_j |v_j| / scale_j."""
    n, _, d = q.shape
    group = nq // nkv
    q = q.double().view(n, nkv, group, d)
    key = torch.arange(keys.shape[1])
    at = pos.view(-1, 1)
    seen = key <= at
    if window:
        seen = seen & (key > at - window)
    # (what is not seen takes no part: not even as zero times a value that is no number)
    k, v = keys.double(), values.double()
    score = torch.einsum("nhgd,hkd->nhgk", q, torch.nan_to_num(k, nan=0.0)) * scale
    score = score + torch.where(k.isnan().any(-1) | v.isnan().any(-1), torch.nan, 0.0).view(1, nkv, 1, -1)
    score = torch.where(seen.view(n, 1, 1, -1), score, -torch.inf)
    reach = (torch.einsum("nhgd,hkd->nhgk", q.abs(), torch.nan_to_num(k, nan=0.0).abs()) * scale)
    reach = torch.where(seen.view(n, 1, 1, -1), reach, 0.0).amax(-1, keepdim=True)
    p = torch.softmax(score, dim=-1)
    p = torch.where(seen.any(-1).view(n, 1, 1, 1), p, 0.0)
    v = torch.nan_to_num(v, nan=0.0)
    out, spread = torch.einsum("nhgk,hkd->nhgd", p, v), torch.einsum("nhgk,hkd->nhgd", p, v.abs())
    three = out.reshape(n, nq, d), spread.reshape(n, nq, d), reach.reshape(n, nq, 1)
    if value_scales is None:
        return three
    s = torch.nan_to_num(value_scales, nan=0.0)
    payload = torch.where(s.unsqueeze(-1) > 0, v.abs() / s.unsqueeze(-1), 0.0)
    beside = torch.nan_to_num(p * s.view(1, nkv, 1, -1), nan=0.0).amax(-1, keepdim=True) * torch.einsum("nhgk,hkd->nhgd", seen.view(n, 1, 1, -1).expand(p.shape).double(), payload)
    return (*three, beside.reshape(n, nq, d))


def step(new, past, page_size, device="cuda:0", *, seed=0, spare=2, shuffled=True):
    """A step's description (ctx, group) as the engine's layout gives it, with every request's pages scattered, and the number of pages."""
    totals = [n + p for n, p in zip(new, past)]
    need = [-(-t // page_size) for t in totals]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 91)).tolist() if shuffled else list(range(pages))
    width = (max(need) + 3) // 4 * 4
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    pos = [p + i for n, p in zip(new, past) for i in range(n)]
    owner = [r for r, n in enumerate(new) for _ in range(n)]
    slots = [table[r][p // page_size] * page_size + p % page_size for r, p in zip(owner, pos)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    arrays, layout = ops.attention_step_layout(list(new))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    ctx = SimpleNamespace(num_tokens=sum(new), num_requests=len(new), positions=ints(pos), request_of=ints(owner), cu_q=ints(cu), kv_len=ints(totals),
                          status=torch.zeros(1, dtype=torch.int32, device=device), host_q_lens=list(new), host_kv_lens=totals, max_q_len=max(new),
                          max_kv_len=max(totals), extras={f"attention.{k}": ints(v) for k, v in arrays.items()}, layout={"attention": layout})
    group = SimpleNamespace(block_table=ints(table), slot_mapping=ints(slots), page_size=page_size, max_pages=width)
    return ctx, group, pages


def random_cache(pages, heads, page_size, d, gen, device="cuda:0", low=118, high=123):
    blocks = page_size // BLOCK
    payload = lambda *shape: (torch.randn(shape, generator=gen) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).to(device)
    scale = lambda: torch.randint(low, high, (pages, heads, blocks), generator=gen, dtype=torch.uint8).to(device).view(torch.float8_e8m0fnu)
    return ops.PagedE4M3(payload(pages, heads, page_size, d), payload(pages, heads, blocks, d, BLOCK), scale(), scale())


def rows_of(table_row, total, page_size):
    """(page, place in it) of a request's first `total` tokens."""
    at = torch.arange(total)
    return table_row.cpu().long()[at // page_size], at % page_size
