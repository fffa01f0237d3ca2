"""The 4-bit key/value cache's operators as a serving program calls them, beside
their plain forms.

  tables     block tables, slots and positions of one scheduling step, from the
             requests' cached and new lengths and a ring of free pages
  append     keys and values quantised into 4-bit pages at their slots, and the
             same slots read back as the values that the codes stand for
  attention  grouped-query attention over the pages: single tokens, drafted
             tokens, and prompt chunks

A page of one kv head is a block of bytes: the codes of page_size keys, the
codes of page_size values (head_dim / 2 bytes a token, the lower column in the
low nibble), then the keys' scales and the values' scales, one per token.  INT4:
fp16 scale = absmax / 7, value (code - 8) * scale; NF4: fp32 absmax, value
table[code] * absmax.  The cache is uint8 [pages][kv_heads][block bytes].
"""
import math
import os
import sys

import numpy as np
import torch

own = False

NF4 = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
       -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
       0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DEVICE = "cuda"


# ---- cases --------------------------------------------------------------------

def tables_case(requests, cached, new, page, **more):
    return dict(op="tables", requests=requests, cached_lo=cached[0], cached_hi=cached[1], new_lo=new[0], new_hi=new[1],
                page=page, **more)


def append_case(fmt, dtype, tokens, kv_heads, head_dim, page, **more):
    return dict(op="append", fmt=fmt, dtype=dtype, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, page=page,
                **more)


def attention_case(fmt, dtype, heads, kv_heads, head_dim, page, requests, cached, new, window=0, **more):
    """`requests` with `cached` = (fewest, most) tokens in the cache before the step and `new` tokens in it."""
    return dict(op="attention", fmt=fmt, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                requests=requests, cached_lo=cached[0], cached_hi=cached[1], new_lo=new[0], new_hi=new[1],
                window=window, **more)


def listed():
    return [
        # one decode step of a small batch: a few hundred integers, so what it costs is latency
        tables_case(48, (100, 4000), (1, 1), 16, name="tables decode 48"),
        # a step that admits prompts beside running requests: 175 thousand slots, some requests without new tokens
        tables_case(700, (0, 3000), (0, 500), 32, name="tables prompts 700"),
        # a decode step's keys and values of one layer, 8 kv heads x 128
        append_case("int4", "fp16", 64, 8, 128, 16, name="append decode int4"),
        # packed prompts of one layer in bf16, 4 kv heads x 128: bandwidth
        append_case("nf4", "bf16", 20011, 4, 128, 32, name="append prompts nf4"),
        # 64-wide heads straight from a projection's fp32 rows
        append_case("int4", "fp32", 6007, 12, 64, 64, name="append prompts int4 64"),
        # one user, a short conversation: the smallest attention call, latency
        attention_case("int4", "fp16", 28, 4, 128, 16, 1, (776, 776), (1, 1), name="decode one"),
        # a full serving batch at 8k tokens, 64 heads over 8: cache bandwidth
        attention_case("int4", "fp16", 64, 8, 128, 64, 32, (8191, 8191), (1, 1), name="decode 32x8k int4"),
        # many requests of every length from 1 to 6000, 64-wide heads, small pages
        attention_case("nf4", "bf16", 32, 8, 64, 16, 96, (0, 5999), (1, 1), name="decode ragged nf4 64"),
        # one request with a very long context: the cache has to be split over the whole GPU
        attention_case("nf4", "fp16", 64, 8, 128, 64, 1, (131070, 131070), (1, 1), name="decode one 131k nf4"),
        # drafted tokens checked in one pass: 5 queries a request
        attention_case("int4", "fp16", 28, 4, 128, 32, 24, (2500, 5500), (5, 5), name="drafts 24x5 int4"),
        # a chunk of a long prompt behind 6000 cached tokens: products
        attention_case("int4", "fp16", 28, 4, 128, 64, 1, (6000, 6000), (2048, 2048), name="prompt chunk int4"),
        # several prompts packed into one step, nothing cached, odd lengths
        attention_case("nf4", "bf16", 64, 8, 128, 32, 5, (0, 0), (200, 1500), name="prompts packed nf4"),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))

    op = rng.choice(("tables", "append", "append", "attention", "attention", "attention", "attention"))
    fmt, page = rng.choice(("int4", "nf4")), rng.choice((16, 32, 64))
    if op == "tables":
        n = spread(1, 700)
        new = (1, 1) if rng.random() < 0.4 else (0, spread(2, max(2, 150000 // n)))
        return tables_case(n, (spread(1, 500) - 1, spread(500, 6000)), new, page)
    kv_heads, head_dim = rng.choice((1, 2, 4, 8, 12)), rng.choice((64, 128, 128))
    if op == "append":
        return append_case(fmt, rng.choice(("fp16", "bf16", "fp32")), spread(1, 40_000_000 // (kv_heads * head_dim * 4)),
                           kv_heads, head_dim, page)
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    kind = rng.choice(("decode", "decode", "drafts", "prompt"))
    limit = 2.4e8                       # bytes of cache
    flops = 1.2e11
    while True:
        n = spread(1, 128) if kind != "prompt" else spread(1, 12)
        hi = spread(1, 131072 if n < 4 else 16384)
        cached = (hi, hi) if rng.random() < 0.3 else (rng.randrange(hi + 1), hi)
        if kind == "decode":
            new = (1, 1)
        elif kind == "drafts":
            new = (rng.choice((0, 2, 3)), rng.randrange(3, 9))
        else:
            new = (rng.randrange(1, 40), spread(40, 2500))
        window = spread(16, 8192) if rng.random() < 0.25 else 0
        c = attention_case(fmt, rng.choice(("fp16", "bf16")), group * kv_heads, kv_heads, head_dim, page, n, cached, new, window)
        w = work(c)
        full = sum(a + b for a, b in zip(*lengths(c))) * kv_heads * head_dim     # what the plain form holds in 32 bits
        rows = n * max(lengths(c)[1]) * group * kv_heads * (cached[1] + new[1])
        if w["bytes"] < limit and w["flops"] < flops and full < 3.5e8 and n * (cached[1] + new[1]) * kv_heads * head_dim < 7e8 and rows < 1.5e9:
            return c


def lengths(case):
    """The requests' cached and new lengths, spread evenly between their bounds in an order that is not sorted."""
    def between(lo, hi, step):
        return [lo + int((hi - lo + 1) * math.modf((r + 1) * step)[0]) for r in range(case["requests"])]

    return between(case["cached_lo"], case["cached_hi"], 0.6180339887), between(case["new_lo"], case["new_hi"], 0.7548776662)


def code_bytes(case):
    """(bytes of a token's codes, bytes of its scale) in one kv head, keys or values."""
    return case["head_dim"] // 2, 2 if case["fmt"] == "int4" else 4


def work(case):
    if case["op"] == "tables":
        cached, new = lengths(case)
        pages = [-(-(a + b) // case["page"]) for a, b in zip(cached, new)]
        held = [-(-a // case["page"]) for a in cached]
        taken = sum(pages) - sum(held)
        # lengths in and out, starts out, free pages in, table entries out, one old page at most in, slots and positions out
        return {"bytes": 4 * (4 * case["requests"] + 2 * taken + 2 * sum(new)), "flops": 0}
    if case["op"] == "append":
        n = case["tokens"] * case["kv_heads"]
        codes, scale = code_bytes(case)
        item = DTYPES[case["dtype"]].itemsize
        # keys and values in, codes and scales out and in again, fp32 values out; a division's worth of work each
        return {"bytes": 2 * n * (case["head_dim"] * (item + 4) + 2 * (codes + scale)) + 8 * case["tokens"],
                "flops": 2 * n * case["head_dim"] * 4}
    cached, new = lengths(case)
    read = pairs = 0
    for c, n in zip(cached, new):
        if n == 0:
            continue
        w = case["window"]
        read += c + n if not w else min(c + n, w + n - 1)
        pairs += n * c + n * (n + 1) // 2 if not w else sum(min(w, c + i + 1) for i in range(n))
    codes, scale = code_bytes(case)
    return {"bytes": 2 * read * case["kv_heads"] * (codes + scale) + 4 * sum(new) * case["heads"] * case["head_dim"]
            + 4 * (read // case["page"] + 2 * case["requests"]),
            "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ---- what a program has in hand --------------------------------------------------

def generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = generator(seed)
    state = dict(case=case)
    if case["op"] == "append":
        t, h, d, page = case["tokens"], case["kv_heads"], case["head_dim"], case["page"]
        pages = -(-t // page) + 3
        # keys and values are column slices of one fused projection's rows
        rows = torch.randn((t, 2 * h * d), generator=g, device=DEVICE)
        rows *= torch.exp(0.5 * torch.randn((t, 1), generator=g, device=DEVICE))
        rows = rows.to(DTYPES[case["dtype"]])
        state.update(k=rows[:, : h * d].view(t, h, d), v=rows[:, h * d:].view(t, h, d),
                     slots=torch.randperm(pages * page, generator=g, device=DEVICE)[:t].to(torch.int32),
                     blocks=torch.zeros((pages, h, page * 2 * sum(code_bytes(case))), dtype=torch.uint8, device=DEVICE),
                     k_out=torch.empty((t, h, d), device=DEVICE), v_out=torch.empty((t, h, d), device=DEVICE))
        return state
    cached, new = lengths(case)
    page = case["page"]
    need = [-(-(a + b) // page) for a, b in zip(cached, new)]
    total = sum(new)
    ints = dict(dtype=torch.int32, device=DEVICE)
    need_t = torch.tensor(need, device=DEVICE)
    start = torch.cumsum(need_t, 0) - need_t
    width = max(need + [1])
    column = torch.arange(width, device=DEVICE)
    pages = sum(need) + 5
    order = torch.randperm(pages, generator=g, device=DEVICE)
    where = start[:, None] + column[None, :]
    if case["op"] == "tables":
        # the pages that the requests hold already, and a ring of the others, read from some place in its middle
        held = torch.tensor([-(-a // page) for a in cached], device=DEVICE)
        tables = torch.where(column[None, :] < held[:, None], order[where.clamp(max=pages - 1)], -1).to(torch.int32)
        free = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        head = int(torch.randint(pages, (1,), generator=torch.Generator().manual_seed(seed)))
        room = -(-max(total, 1) // 64) * 64                          # slots are laid out for a step of this many tokens
        state.update(tables=tables, cached=torch.tensor(cached, **ints), new=torch.tensor(new, **ints), free_pages=free,
                     free_state=torch.tensor([head, pages - 2, 0], **ints), room=room)
        return state
    state["tables"] = torch.where(column[None, :] < need_t[:, None], order[where.clamp(max=pages - 1)], -1).to(torch.int32)
    state["ctx_len"] = torch.tensor([a + b for a, b in zip(cached, new)], **ints)
    state["q_starts"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), **ints)
    state["max_q"] = max(new)
    state["longest"] = max(a + b for a, b in zip(cached, new))
    h, d = case["kv_heads"], case["head_dim"]
    # keys with a few strong columns, values plain; both with tokens of unlike size
    parts, scales = [], []
    for strong in (True, False):
        x = torch.randn((pages, h, page, d), generator=g, device=DEVICE)
        if strong:
            x *= 1 + 2 * (torch.rand((1, h, 1, d), generator=g, device=DEVICE) > 0.95)
        x *= torch.exp(0.25 * torch.randn((pages, h, page, 1), generator=g, device=DEVICE))
        amax = x.abs().amax(-1, keepdim=True)
        if case["fmt"] == "int4":
            s = (amax / 7).half()
            codes = torch.round(x / s.float()).add_(8).clamp_(0, 15).to(torch.uint8)
        else:
            s = amax
            t = torch.tensor(NF4, device=DEVICE)
            codes = torch.bucketize(x / s, (t[1:] + t[:-1]) / 2, out_int32=True).to(torch.uint8)
        del x
        parts.append((codes[..., 0::2] | codes[..., 1::2] << 4).view(pages, h, -1))
        scales.append(s.view(torch.uint8).view(pages, h, -1))
    state["blocks"] = torch.cat(parts + scales, -1).contiguous()
    q = torch.randn((total, case["heads"], d), generator=g, device=DEVICE)
    state["q"] = q.to(DTYPES[case["dtype"]])
    state["out"] = torch.empty_like(state["q"])
    return state


def parts_of(case, blocks):
    """Views of [..., block bytes]: key and value codes [..., page, head_dim / 2], key and value scales in fp32."""
    page = case["page"]
    codes, scale = code_bytes(case)
    lead = blocks.shape[:-1]
    k, v, ks, vs = torch.split(blocks, [page * codes, page * codes, page * scale, page * scale], -1)
    kind = torch.float16 if case["fmt"] == "int4" else torch.float32
    return (k.reshape(*lead, page, codes), v.reshape(*lead, page, codes),
            ks.contiguous().view(kind).float(), vs.contiguous().view(kind).float())


# ---- one pass ---------------------------------------------------------------------

def run(state):
    return (run_own if own else run_plain)(state)


def run_own(state):
    case = state["case"]
    if "lib" not in state:          # the program's imports and its handle of the cache
        at = os.path.join(os.getcwd(), "int4-gemv_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import b4gemv
        state["lib"] = b4gemv
        if case["op"] != "tables":
            fmt = b4gemv.KV_INT4 if case["fmt"] == "int4" else b4gemv.KV_NF4
            state["cache"] = b4gemv.KVCache(state["blocks"], fmt, case["page"], case["head_dim"])
    lib = state["lib"]
    if case["op"] == "tables":
        step = lib.kv_tables(case["page"], state["tables"], state["cached"], state["new"], state["free_pages"],
                             state["free_state"], state["room"])
        return dict(tables=state["tables"], ctx_len=step.ctx_len, q_starts=step.q_starts, slots=step.slots,
                    positions=step.positions, free_state=step.free_state)
    if case["op"] == "append":
        lib.kv_append(state["cache"], state["k"], state["v"], state["slots"])
        k, v = lib.kv_read(state["cache"], state["slots"], state["k_out"], state["v_out"])
        return dict(k=k, v=v)
    return lib.kv_attention(state["cache"], state["q"], state["tables"], state["ctx_len"], state["q_starts"],
                            state["max_q"], window=case["window"], out=state["out"])


def run_plain(state):
    return dict(tables=plain_tables, append=plain_append, attention=plain_attention)[state["case"]["op"]](state)


def plain_tables(state):
    page, room = state["case"]["page"], state["room"]
    tables, cached, new = state["tables"], state["cached"].long(), state["new"].long()
    free, fs = state["free_pages"], state["free_state"].long()
    width = tables.shape[1]
    ctx = cached + new
    held, need = (cached + page - 1) // page, (ctx + page - 1) // page
    fresh = need - held
    first = torch.cumsum(fresh, 0) - fresh
    q_starts = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    column = torch.arange(width, device=tables.device)
    n = first[:, None] + column - held[:, None]
    page_of = torch.where(n < fs[1], free[(fs[0] + n) % free.shape[0]].long(), -1)
    tables = torch.where((column >= held[:, None]) & (column < need[:, None]), page_of, tables.long())
    token = torch.arange(room, device=tables.device)
    r = torch.searchsorted(q_starts[1:], token, right=True).clamp(max=new.shape[0] - 1)
    position = cached[r] + token - q_starts[r]
    at = tables[r, (position // page).clamp(max=width - 1)]
    there = token < q_starts[-1]
    taken = torch.minimum(fresh.sum(), fs[1])
    state_out = torch.stack([(fs[0] + taken) % free.shape[0], fs[1] - taken, fresh.sum() - taken])
    slots = torch.where(there & (at >= 0), at * page + position % page, -1)
    return dict(tables=tables.int(), ctx_len=ctx.int(), q_starts=q_starts.int(), slots=slots.int(),
                positions=torch.where(there, position, 0).int(), free_state=state_out.int())


def plain_quantise(case, x):
    """Codes (bytes of two) and scales, as bytes, of x [tokens, kv_heads, head_dim]."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    if case["fmt"] == "int4":
        s = torch.where(amax > 0, amax / 7, 1.0).half()
        y = x / s.float()
        whole = torch.trunc(y)
        codes = (whole + torch.sign(y) * ((y - whole).abs() >= 0.5) + 8).clamp(0, 15).to(torch.uint8)
    else:
        s = torch.where(amax > 0, amax, 1.0)
        d = ((x / s)[..., None] - torch.tensor(NF4, device=x.device)).abs()
        nearest = torch.where(d == d.amin(-1, keepdim=True), torch.arange(16, device=x.device), 16)
        codes = nearest.amin(-1).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, s.contiguous().view(torch.uint8)


def plain_values(case, codes, scales):
    """fp32 values of codes [..., head_dim / 2] bytes with one fp32 scale for each token."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    if case["fmt"] == "int4":
        return (c.float() - 8) * scales[..., None]
    return torch.tensor(NF4, device=c.device)[c.int()] * scales[..., None]


def plain_append(state):
    case, blocks, slots = state["case"], state["blocks"], state["slots"].long()
    page = case["page"]
    codes, scale = code_bytes(case)
    kb, ks = plain_quantise(case, state["k"])
    vb, vs = plain_quantise(case, state["v"])
    at, row = slots // page, slots % page
    heads = torch.arange(case["kv_heads"], device=blocks.device)[None, :, None]

    def places(base, size):
        return at[:, None, None], heads, base + (row * size)[:, None, None] + torch.arange(size, device=blocks.device)

    bases = [(0, codes), (page * codes, codes), (2 * page * codes, scale), (2 * page * codes + page * scale, scale)]
    where = [places(*b) for b in bases]
    blocks[where[0]] = kb
    blocks[where[1]] = vb
    blocks[where[2]] = ks
    blocks[where[3]] = vs
    kind = torch.float16 if case["fmt"] == "int4" else torch.float32
    return dict(k=plain_values(case, blocks[where[0]], blocks[where[2]].view(kind).squeeze(-1).float()),
                v=plain_values(case, blocks[where[1]], blocks[where[3]].view(kind).squeeze(-1).float()))


def plain_attention(state):
    case, q, ctx, starts = state["case"], state["q"], state["ctx_len"].long(), state["q_starts"].long()
    b, h, d, most = ctx.shape[0], case["kv_heads"], case["head_dim"], max(state["max_q"], 1)
    group, total = case["heads"] // h, q.shape[0]
    kc, vc, ks, vs = parts_of(case, state["blocks"][state["tables"].long().clamp(min=0)])     # [b, pages, h, page, ...]
    k, v = (plain_values(case, c, s).transpose(1, 2).reshape(b, h, -1, d) for c, s in ((kc, ks), (vc, vs)))
    n = starts[1:] - starts[:-1]
    row = torch.arange(most, device=q.device)
    # the requests' queries, padded to the longest, grouped by the kv head that they share
    at = (starts[:-1, None] + row).clamp(max=total - 1)
    wide = q.float()[at].view(b, most, h, group, d).permute(0, 2, 3, 1, 4).reshape(b, h, group * most, d)
    s = torch.matmul(wide, k.transpose(-1, -2)).mul_(d ** -0.5).view(b, h, group, most, -1)
    key = torch.arange(k.shape[2], device=q.device)
    own_key = ctx[:, None] - n[:, None] + row                                                  # the query's own place
    seen = (key <= own_key[:, :, None]) & (key < ctx[:, None, None])
    if case["window"]:
        seen &= key > own_key[:, :, None] - case["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)))
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30)).view(b, h, group * most, -1)
    o = torch.matmul(p, v).view(b, h, group, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, case["heads"], d)
    token = torch.arange(total, device=q.device)
    r = torch.searchsorted(starts[1:], token, right=True)
    return o[r, token - starts[r]].to(q.dtype)


# ---- from the definitions, in 64 bits -----------------------------------------------

def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return dict(k=exact_rounded(case, s["k"]), v=exact_rounded(case, s["v"]))
    q, h, d, page = s["q"].double(), case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // h
    kb, vb, ks, vs = parts_of(case, s["blocks"])
    out = torch.zeros_like(q)
    starts, ctx = s["q_starts"].tolist(), s["ctx_len"].tolist()
    for r in range(case["requests"]):
        n, length = starts[r + 1] - starts[r], ctx[r]
        if n == 0:
            continue
        ids = s["tables"][r, : -(-length // page)].long()
        for i in range(h):
            k, v = (exact_values(case, codes[ids, i].reshape(-1, d // 2)[:length], scale[ids, i].reshape(-1)[:length])
                    for codes, scale in ((kb, ks), (vb, vs)))
            x = q[starts[r]: starts[r + 1], i * group: (i + 1) * group].reshape(n * group, d)
            a = x @ k.T / math.sqrt(d)
            last = torch.arange(length - n, length, device=a.device).repeat_interleave(group)[:, None]
            place = torch.arange(length, device=a.device)[None, :]
            a[(place > last) | ((place <= last - case["window"]) if case["window"] else (place < 0))] = -math.inf
            out[starts[r]: starts[r + 1], i * group: (i + 1) * group] = (torch.softmax(a, -1) @ v).view(n, group, d)
    return out


def exact_values(case, codes, scale):
    low, high = (codes % 16).long(), (codes // 16).long()
    levels = torch.arange(-8, 8, device=codes.device).double() if case["fmt"] == "int4" else \
        torch.tensor(NF4, dtype=torch.float64, device=codes.device)
    values = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64, device=codes.device)
    values[:, 0::2], values[:, 1::2] = levels[low], levels[high]
    return values * scale.double()[:, None]


def exact_rounded(case, x):
    """x [tokens, kv_heads, head_dim] replaced by the nearest values that a token's scale allows."""
    x = x.double()
    top = x.abs().max(-1, keepdim=True).values
    top[top == 0] = 1 if case["fmt"] == "nf4" else 7
    if case["fmt"] == "int4":
        step = (top / 7).half().double()
        y = x / step
        return torch.clamp(torch.sign(y) * torch.floor(y.abs() + 0.5), -8, 7) * step
    levels = torch.tensor(NF4, dtype=torch.float64, device=x.device)
    y = (x / top).contiguous()
    right = torch.searchsorted(levels, y).clamp(1, 15)
    nearer = (y - levels[right - 1]) <= (levels[right] - y)
    return levels[right - nearer.long()] * top
