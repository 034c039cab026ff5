"""The operators of serving in few bits that are measured: what a decode step reads, keys and values in 8 bits
and weights in 4.

A case's `kind`:
  append     a step's projected queries, keys and values: head norm and rotation, the queries handed on, the
             keys and values rounded into a paged cache of 8 bits with a scale for each block of 16 tokens and head
  attend     attention of a step's queries over that cache: single tokens, portions of prompts, or both
  product    x @ W.T with weights in 4 bits and a scale for each group along k

The cache, per layer: `k` float8_e4m3fn [pages, kv heads, page, d] and `v` [pages, kv heads, page / 16, d, 16] (inside a
block of 16 tokens a feature's values lie side by side), `k_scale` and `v_scale` float8_e8m0fnu [pages, kv heads,
page / 16]. What is held is payload * scale. A block's scale is the smallest power of two that brings its largest value to
448 or below; where a later token needs a larger one, the tokens that are there are rounded to it.

The weights: `codes` uint8 [features / 16, k / 128, 16 rows, 4, 4, 4 bytes]: of a row's 128 codes, byte [j][i][.] holds
those of k = 32 i + 8 j .. 32 i + 8 j + 7, as a 32-bit word whose nibble p is the code of k offset 2 p (p < 4) or 2 p - 7; a
code c is held as c + 8. `scales` bfloat16 [features / 16, k / 128, 16, 128 / group]. Rows and k beyond the matrix are
there and do not count.

`new` (tokens each request brings) and `past` (tokens of each request that the cache holds already) as "2048" or "1,1,1".
"""
import math
from types import SimpleNamespace

import torch

own = False

EPS, THETA = 1e-6, 1000000.0
TOKENS = 16                      # of a block with one scale


def _step(kind, new, past, heads=32, kv=8, dim=128, page=16, dtype="bfloat16", window=0, rotary=0, neighbours=False):
    return dict(kind=kind, new=",".join(map(str, new)), past=",".join(map(str, past)), heads=heads, kv=kv, dim=dim, page=page,
                dtype=dtype, window=window, rotary=rotary or dim, neighbours=neighbours)


def _product(rows, features, k, group=128):
    return dict(kind="product", rows=rows, features=features, k=k, group=group)


def _ragged(count, low, high):
    """`count` lengths spread over low .. high in a mixed order."""
    return [low + (high - low) * ((i * 37 + 11) % 64) // 63 for i in range(count)]


def listed():
    named = [
        # a layer of the 8B sizes while it generates for the benchmark's batch of eight
        ("append_decode_8", _step("append", [1] * 8, [2047] * 8)),
        # a prompt of the benchmark's length in one step
        ("append_prefill_2048", _step("append", [2048], [0])),
        # a continuous batch: portions that begin and end inside a block beside requests that generate, on the float32 path
        ("append_ragged_float32", _step("append", [509, 131] + [1] * 13, [1029, 0] + _ragged(13, 70, 2900), 16, 4, 64, 32, "float32")),
        # generating for one user, for eight with a long past, and for a full server whose requests differ
        ("attend_decode_1", _step("attend", [1], [2047])),
        ("attend_decode_8_long", _step("attend", [1] * 8, [16383] * 8)),
        ("attend_decode_64", _step("attend", [1] * 64, _ragged(64, 600, 3500))),
        # a prompt of the benchmark's length, and a continuous batch of portions beside generation
        ("attend_prefill_2048", _step("attend", [2048], [0])),
        ("attend_mixed", _step("attend", [509, 131] + [1] * 13, [1029, 0] + _ragged(13, 70, 2900))),
        # the output projection for one user, gate and up for eight, down for a full server, gate and up of a prompt
        ("product_1", _product(1, 4096, 4096)),
        ("product_8", _product(8, 24576, 4096)),
        ("product_64", _product(64, 4096, 12288, 64)),
        ("product_prefill_2048", _product(2048, 24576, 4096)),
    ]
    return [dict(case, name=name) for name, case in named]


def draw(rng):
    spread = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    kind = rng.choice(["append", "attend", "attend", "product"])
    if kind == "product":
        group = rng.choice([32, 64, 128, 128])
        rows = spread(1, 2048)
        features, k = spread(500, 24576), group * spread(max(2, 512 // group), 12288 // group)
        while rows * features * k > 2048 * 24576 * 4096 * 0.9:
            features = max(500, features // 2)
        return _product(rows, features, k, group)
    kv = rng.choice([1, 4, 8])
    sizes = dict(heads=kv * rng.choice([1, 2, 4, 5, 8]), kv=kv, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 16, 32, 64]))
    if rng.random() < 0.15:          # the float32 path: few tokens
        sizes["dtype"] = "float32"
        new = [spread(1, 60) for _ in range(rng.randint(1, 4))]
        past = [rng.choice([0, rng.randint(1, 1000)]) for _ in new]
    elif rng.random() < 0.5:         # generating
        new = [1] * spread(1, 64)
        longest = spread(64, 16000 if len(new) <= 8 else 3500)
        past = [rng.randint(1, longest) for _ in new]
    else:                            # portions of prompts, perhaps beside requests that generate
        portions = rng.randint(1, 3)
        new = [spread(5, 2048 // portions) for _ in range(portions)]
        past = [rng.choice([0, rng.randint(1, 1500)]) for _ in new]
        if rng.random() < 0.4:
            count = rng.randint(1, 12)
            new, past = new + [1] * count, past + [rng.randint(16, 2000) for _ in range(count)]
    if kind == "attend":
        sizes["window"] = rng.choice([0, 0, 0, rng.randint(20, 1200)])
    else:
        whole = rng.random() < 0.7
        sizes["rotary"], sizes["neighbours"] = (0, False) if whole else (sizes["dim"] // 2, rng.random() < 0.5)
    return _step(kind, new, past, **sizes)


# ---------------------------------------------------------------- inputs, from the seed alone
def _lengths(case):
    return [int(v) for v in case["new"].split(",")], [int(v) for v in case["past"].split(",")]


def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


def _cuda(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _cache(case, pages, normal, uniform):
    kv, dim, page = case["kv"], case["dim"], case["page"]
    blocks = page // TOKENS
    # payloads as rounding normal values leaves them, scales over a few powers of two
    payload = lambda *shape: (normal(*shape) * 110.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    scale = lambda low: (uniform(pages, kv, blocks, low=low, high=low + 4.0).floor().to(torch.uint8)).view(torch.float8_e8m0fnu)
    return dict(k=payload(pages, kv, page, dim), v=payload(pages, kv, blocks, dim, TOKENS), k_scale=scale(119.0), v_scale=scale(118.0))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 29)
    normal = lambda *shape, std=1.0, mean=0.0, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)
    uniform = lambda *shape, low, high: torch.empty(shape, device="cuda").uniform_(low, high, generator=gen)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["kind"] == "product":
        rows, features, k, group = case["rows"], case["features"], case["k"], case["group"]
        tiles, deep = -(-features // 16), -(-k // 128)
        codes = torch.randint(0, 256, (tiles, deep, 16, 4, 4, 4), generator=gen, dtype=torch.uint8, device="cuda")
        scales = uniform(tiles, deep, 16, 128 // group, low=0.002, high=0.008).bfloat16()
        return dict(case=case, x=normal(rows, k, dtype=torch.bfloat16), codes=codes, scales=scales, status=status)

    new, past = _lengths(case)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    dtype, tokens, requests = _dtype(case), sum(new), len(new)
    totals = [n + p for n, p in zip(new, past)]
    need = [-(-t // page) for t in totals]
    pages = sum(need) + 3
    # requests' pages lie between one another's, as they do when the requests came in turns
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5)).tolist()
    width = (max(need) + 3) // 4 * 4
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    positions = [p + i for n, p in zip(new, past) for i in range(n)]
    owner = [r for r, n in enumerate(new) for _ in range(n)]
    slots = [table[r][p // page] * page + p % page for r, p in zip(owner, positions)]
    cache = _cache(case, pages, normal, uniform)
    state = dict(case=case, cache=cache, status=status)
    if case["kind"] == "append":
        half = case["rotary"] // 2
        limit = max(4096, max(totals))
        angle = torch.arange(limit, dtype=torch.float64).view(-1, 1) * THETA ** (-torch.arange(half, dtype=torch.float64) / half)
        # the blocks that the step writes, the first slot it writes of each, and each token's block among them
        blocks, first, block_of = {}, [], []
        for s in slots:
            if s // TOKENS not in blocks:
                blocks[s // TOKENS] = len(blocks)
                first.append(s % TOKENS)
            block_of.append(blocks[s // TOKENS])
        state.update(qkv=normal(tokens, (heads + 2 * kv) * dim, dtype=dtype), q_norm=normal(dim, std=0.1, mean=1.0, dtype=dtype),
                     k_norm=normal(dim, std=0.1, mean=1.0, dtype=dtype), cos=angle.cos().float().cuda(), sin=angle.sin().float().cuda(),
                     positions=_cuda(positions), slots=_cuda(slots), blocks=_cuda(list(blocks), torch.int64), first=_cuda(first, torch.int64),
                     block_of=_cuda(block_of, torch.int64))
        return state
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    # the step's description, as the engine's batch layout gives it: requests of up to four tokens one query at a time, longer
    # ones as portions; lists that would name every token or request are left out
    few = [n <= 4 for n in new] if max(new) > 1 else [True] * requests
    short = [t for r in range(requests) if few[r] for t in range(starts[r], starts[r + 1])]
    long = [r for r in range(requests) if not few[r]]
    lists = {"attention.short_tokens": _cuda(short), "attention.long_rows": _cuda(long)} if short and long else {}
    ctx = SimpleNamespace(num_tokens=tokens, num_requests=requests, positions=_cuda(positions), request_of=_cuda(owner), cu_q=_cuda(starts),
                          kv_len=_cuda(totals), status=status, host_q_lens=new, host_kv_lens=totals, max_q_len=max(new),
                          max_kv_len=max(totals), extras=lists,
                          layout={"attention": dict(num_short_tokens=len(short), num_long_rows=len(long), max_long_q_len=max((new[r] for r in long), default=0))})
    group = SimpleNamespace(block_table=_cuda(table), slot_mapping=_cuda(slots), page_size=page, max_pages=width)
    state.update(ctx=ctx, group=group, q=normal(tokens, heads * dim, dtype=dtype), place=_cuda([i for n in new for i in range(n)], torch.int64))
    return state


# ---------------------------------------------------------------- one pass
def _turned(x, cos, sin, rotary, neighbours):
    """x [..., d] with its first `rotary` elements rotated."""
    head, rest = x[..., :rotary], x[..., rotary:]
    if neighbours:
        a, b = head[..., 0::2], head[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)
    a, b = head[..., :rotary // 2], head[..., rotary // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def _exponents(scale):
    return scale.view(torch.uint8).int() - 127


def _store(rows, payload, scale, state, by_feature):
    """Rounds rows [T, kv, d] into the blocks that the step writes."""
    case = state["case"]
    kv, dim, per_page = case["kv"], case["dim"], case["page"] // TOKENS
    blocks, first, block_of, slots = state["blocks"], state["first"], state["block_of"], state["slots"].long()
    page, part = blocks // per_page, blocks % per_page
    largest = torch.zeros(blocks.shape[0], kv, device="cuda").index_reduce_(0, block_of, rows.abs().amax(-1), "amax")
    mantissa, power = torch.frexp(largest)
    wanted = torch.where(largest > 0, power - 9 + (mantissa > 0.875).int(), torch.full_like(power, -127)).clamp_(min=-127)
    held = _exponents(scale)[page, :, part]
    exponent = torch.where((first > 0).view(-1, 1), torch.maximum(wanted, held), wanted)
    # what the blocks hold already, rounded to the larger scale
    content = payload.view(-1, kv, per_page, dim, TOKENS)[page, :, part] if by_feature else payload.view(-1, kv, per_page, TOKENS, dim)[page, :, part].transpose(-1, -2)
    there = (torch.arange(TOKENS, device="cuda").view(1, -1) < first.view(-1, 1)).view(-1, 1, 1, TOKENS)
    shrunk = torch.ldexp(content.float(), torch.where((first > 0).view(-1, 1), held - exponent, 0).view(-1, kv, 1, 1)).to(torch.float8_e4m3fn)
    content = torch.where(there, shrunk.view(torch.uint8), content.view(torch.uint8))
    # the new tokens
    at = torch.ldexp(rows, -exponent[block_of].unsqueeze(-1)).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    content[block_of, :, :, slots % TOKENS] = at.view(torch.uint8)
    if by_feature:
        payload.view(torch.uint8).view(-1, kv, per_page, dim, TOKENS)[page, :, part] = content
    else:
        payload.view(torch.uint8).view(-1, kv, per_page, TOKENS, dim)[page, :, part] = content.transpose(-1, -2)
    scale.view(torch.uint8)[page, :, part] = (exponent + 127).to(torch.uint8)


def _append(state):
    case, cache = state["case"], state["cache"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    rows = state["qkv"].float().view(-1, heads + 2 * kv, dim)
    cos, sin = (state[name][state["positions"].long()].unsqueeze(1) for name in ("cos", "sin"))
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    turn = lambda x: _turned(x, cos, sin, case["rotary"], case["neighbours"])
    q = turn(norm(rows[:, :heads], state["q_norm"]))
    _store(turn(norm(rows[:, heads:heads + kv], state["k_norm"])), cache["k"], cache["k_scale"], state, False)
    _store(rows[:, heads + kv:], cache["v"], cache["v_scale"], state, True)
    return dict(q=q.reshape(-1, heads * dim).to(_dtype(case)), **cache)


def _attend(state):
    case, ctx, group, cache = state["case"], state["ctx"], state["group"], state["cache"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    requests, most = ctx.num_requests, ctx.max_kv_len
    held = group.block_table[:, :-(-most // page)].long()
    spread = lambda scale: scale.float()[held].transpose(1, 2).flatten(2, 3).repeat_interleave(TOKENS, dim=2)[:, :, :most].unsqueeze(-1)
    keys = cache["k"].float()[held].transpose(1, 2).flatten(2, 3)[:, :, :most] * spread(cache["k_scale"])                  # [B, kv, keys, d]
    values = cache["v"].float()[held].permute(0, 2, 1, 3, 5, 4).flatten(2, 4)[:, :, :most] * spread(cache["v_scale"])
    at = (ctx.request_of.long(), state["place"])
    q = torch.zeros(requests, ctx.max_q_len, heads * dim, device="cuda")
    q[at] = state["q"].float()
    q = q.view(requests, ctx.max_q_len, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)                                   # [B, kv, group, q, d]
    position = torch.full((requests, ctx.max_q_len), -1, device="cuda", dtype=torch.int64)
    position[at] = ctx.positions.long()
    key = torch.arange(most, device="cuda")
    seen = key <= position.unsqueeze(-1)
    if case["window"]:
        seen &= key > position.unsqueeze(-1) - case["window"]
    score = torch.einsum("bkgqd,bknd->bkgqn", q, keys) * dim ** -0.5
    score = score.masked_fill(~seen.view(requests, 1, 1, ctx.max_q_len, most), -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp_(min=-3.0e38))
    out = torch.einsum("bkgqn,bknd->bkgqd", weight / weight.sum(-1, keepdim=True).clamp_(min=1e-38), values)
    return out.permute(0, 3, 1, 2, 4).reshape(requests, ctx.max_q_len, heads * dim)[at].to(_dtype(case))


def _weights(state):
    case = state["case"]
    codes = state["codes"]
    tiles, deep = codes.shape[:2]
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)            # [.., j, i, nibble p of a word]
    order = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device="cuda")                  # k offset -> nibble
    c = nibbles[..., order].float() - 8.0
    c = c.transpose(3, 4).reshape(tiles, deep, 16, 128 // case["group"], case["group"])      # k = 32 i + 8 j + offset
    c = (c * state["scales"].float().unsqueeze(-1)).flatten(3)
    return c.transpose(1, 2).reshape(tiles * 16, deep * 128)[:case["features"], :case["k"]]


def run(state):
    case = state["case"]
    if own:
        from vosti_b200 import ops
        if case["kind"] == "product":
            if "handle" not in state:
                state["handle"] = ops.Int4Weight(state["codes"], state["scales"], (case["features"], case["k"]))
            return ops.gemm_int4(state["x"], state["handle"], state["status"])
        if "handle" not in state:
            state["handle"] = ops.PagedE4M3(**state["cache"])
        sizes = dict(nq=case["heads"], nkv=case["kv"], head_dim=case["dim"])
        if case["kind"] == "append":
            q = ops.qkv_post_e4m3(state["qkv"], state["handle"], q_norm_w=state["q_norm"], k_norm_w=state["k_norm"], eps=EPS, cos=state["cos"],
                                  sin=state["sin"], positions=state["positions"], slot_mapping=state["slots"], status=state["status"],
                                  rotary_dim=case["rotary"], interleaved=case["neighbours"], **sizes)
            return dict(q=q, **state["cache"])
        return ops.attention_e4m3(state["ctx"], state["q"], state["handle"], state["group"], scale=case["dim"] ** -0.5, window=case["window"], **sizes)
    if case["kind"] == "product":
        return (state["x"].float() @ _weights(state).T).to(torch.bfloat16)
    return _append(state) if case["kind"] == "append" else _attend(state)


# ---------------------------------------------------------------- the definition in 64 bits
def _held(payload):
    """The numbers that float8_e4m3fn bytes stand for: sign, 4 bits of exponent (bias 7), 3 of mantissa."""
    b = payload.view(torch.uint8).double()
    sign, e, m = torch.floor(b / 128), torch.floor(b / 8) % 16, b % 8
    return (1 - 2 * sign) * torch.where(e > 0, (8 + m) * 2.0 ** (e - 10), m * 2.0 ** -9)


def _scales(scale):
    return 2.0 ** (scale.view(torch.uint8).double() - 127)


def _to_e4m3(x):
    """The nearest number of that format, ties to an even last bit; at most 448."""
    grid = 2.0 ** torch.clamp(torch.floor(torch.log2(x.abs().clamp(min=1e-300))), min=-6.0) / 8
    return torch.clamp(torch.round(x / grid) * grid, -448.0, 448.0)


def _exact_append(case, s):
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    per_page, rotary = page // TOKENS, case["rotary"]
    x = s["qkv"].double().view(-1, heads + 2 * kv, dim)
    pos = s["positions"].long()
    pairs = torch.arange(rotary // 2, device="cuda")
    ia, ib = (2 * pairs, 2 * pairs + 1) if case["neighbours"] else (pairs, pairs + rotary // 2)
    cos, sin = s["cos"].double()[pos].unsqueeze(1), s["sin"].double()[pos].unsqueeze(1)

    def turned(h, w):
        h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / dim + EPS) * w.double()
        y = h.clone()
        y[..., ia] = h[..., ia] * cos - h[..., ib] * sin
        y[..., ib] = h[..., ib] * cos + h[..., ia] * sin
        return y
    q = turned(x[:, :heads], s["q_norm"])
    out = dict(q=q.reshape(-1, heads * dim))
    slots = s["slots"].tolist()
    runs, t = [], 0
    while t < len(slots):
        n = 1
        while t + n < len(slots) and slots[t + n] // TOKENS == slots[t] // TOKENS:
            n += 1
        runs.append((t, n))
        t += n
    for name, rows in (("k", turned(x[:, heads:heads + kv], s["k_norm"])), ("v", x[:, heads + kv:])):
        scale = _scales(s["cache"][name + "_scale"])
        content = _held(s["cache"][name]).view(-1, kv, per_page, dim, TOKENS) if name == "v" else _held(s["cache"][name]).view(-1, kv, per_page, TOKENS, dim).transpose(-1, -2).contiguous()
        for t, n in runs:
            page_at, part, at = slots[t] // page, slots[t] % page // TOKENS, slots[t] % TOKENS
            fresh = rows[t:t + n].permute(1, 2, 0)                                   # [kv, d, n]
            most = fresh.abs().amax((1, 2))
            power = torch.where(most > 0, torch.ceil(torch.log2(most.clamp(min=1e-300) / 448)), torch.full_like(most, -127.0)).clamp(min=-127.0)
            wanted = 2.0 ** power
            if at:
                wanted = torch.maximum(wanted, scale[page_at, :, part])
                block = content[page_at, :, part, :, :at]
                content[page_at, :, part, :, :at] = _to_e4m3(block * (scale[page_at, :, part] / wanted).view(-1, 1, 1))
            content[page_at, :, part, :, at:at + n] = _to_e4m3(fresh / wanted.view(-1, 1, 1))
            scale[page_at, :, part] = wanted
        out[name] = content if name == "v" else content.transpose(-1, -2).reshape(-1, kv, page, dim)
        out[name + "_scale"] = scale
    return out


def _exact_attend(case, s):
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    new, past = _lengths(case)
    out, t = [], 0
    for r, (n, p) in enumerate(zip(new, past)):
        total = n + p
        pages = s["group"].block_table[r, :-(-total // page)].long()
        each = lambda name: _scales(s["cache"][name][pages]).repeat_interleave(TOKENS, dim=2).unsqueeze(-1)          # [pages, kv, page, 1]
        keys = (_held(s["cache"]["k"][pages]) * each("k_scale")).transpose(0, 1).flatten(1, 2)[:, :total]
        values = (_held(s["cache"]["v"][pages]).transpose(-1, -2).flatten(2, 3) * each("v_scale")).transpose(0, 1).flatten(1, 2)[:, :total]
        q = s["q"][t:t + n].double().view(n, kv, heads // kv, dim)
        at, key = torch.arange(p, total, device="cuda").view(-1, 1), torch.arange(total, device="cuda")
        hidden = key > at
        if case["window"]:
            hidden = hidden | (key <= at - case["window"])
        rows = []
        for h in range(kv):
            score = torch.einsum("qgd,nd->gqn", q[:, h], keys[h]) / math.sqrt(dim)
            rows.append(torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ values[h])                   # [group, q, d]
        out.append(torch.stack(rows).permute(2, 0, 1, 3).reshape(n, heads * dim))
        t += n
    return torch.cat(out)


def _exact_product(case, s):
    features, k, group = case["features"], case["k"], case["group"]
    column = torch.arange(k, device="cuda")
    block, inside = column // 128, column % 128
    i, j, offset = inside // 32, inside % 32 // 8, inside % 8
    nibble = torch.where(offset % 2 == 0, offset // 2, offset // 2 + 4)
    part = inside // group
    x, out = s["x"].double(), []
    for f0 in range(0, features, 4096):
        row = torch.arange(f0, min(f0 + 4096, features), device="cuda").view(-1, 1)
        byte = s["codes"][row // 16, block, row % 16, j, i, nibble // 2].int()
        code = torch.where(nibble % 2 == 0, byte % 16, byte // 16) - 8
        out.append(x @ (code.double() * s["scales"].double()[row // 16, block, row % 16, part]).T)
    return torch.cat(out, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "product": _exact_product}[case["kind"]](case, state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "product":
        rows, features, k = case["rows"], case["features"], case["k"]
        return {"bytes": features * k // 2 + features * (k // case["group"]) * 2 + 2 * rows * (k + features), "flops": 2 * rows * features * k}
    new, past = _lengths(case)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    size, tokens = (4 if case["dtype"] == "float32" else 2), sum(new)
    if case["kind"] == "append":
        blocks = sum((p % TOKENS + n + TOKENS - 1) // TOKENS for n, p in zip(new, past))
        tables = len({p + i for n, p in zip(new, past) for i in range(n)}) * case["rotary"] * 4
        return {"bytes": tokens * (2 * heads + 2 * kv) * dim * size + tokens * 2 * kv * dim + 2 * kv * blocks + tables, "flops": tokens * (heads + 2 * kv) * dim * 10}
    window = case["window"]
    first = lambda at: max(0, at - window + 1) if window else 0
    read = sum(p + n - first(p) for n, p in zip(new, past))
    pairs = sum(at + 1 - first(at) for n, p in zip(new, past) for at in range(p, p + n))
    return {"bytes": 2 * tokens * heads * dim * size + read * kv * (2 * dim + 2 / TOKENS), "flops": 4 * pairs * heads * dim}
