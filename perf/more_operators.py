"""Operators of a layer over the 4-bit key/value cache whose queries read a choice of
its pages, as a serving program calls them, beside their plain forms.

  append     the rotation of queries and keys by their positions (one axis or several)
             on the way into the 4-bit pages, and the same slots read back
  select     the boxes around the keys of the pages that a step completed, then for
             every query and kv head the pages whose boxes bound its scores highest
  attention  attention of every query over its own list of pages

A page of one kv head is a block of bytes: the codes of page_size keys, the codes
of page_size values (head_dim / 2 bytes a token, the lower column in the low
nibble), then the keys' scales and the values' scales, one per token.  INT4: fp16
scale = absmax * (1 / 7), value (code - 8) * scale; NF4: fp32 absmax, value
table[code] * absmax.  The cache is uint8 [pages][kv_heads][block bytes].

A page's box of one kv head: head_dim bytes of its keys' column maxima and
head_dim of their minima, as int8 in units of an fp32 scale (absmax * (1 / 127))
that follows them, and 12 bytes of zeros.
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

def append_case(fmt, dtype, tokens, heads, kv_heads, head_dim, page, rotated, axes, adjacent, far, **more):
    """`rotated` columns of a head turn, in pairs of neighbours or of halves, by positions below `far` on `axes` axes."""
    return dict(op="append", fmt=fmt, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                rotated=rotated, axes=axes, adjacent=adjacent, far=far, **more)


def select_case(fmt, dtype, heads, kv_heads, head_dim, page, requests, cached, new, keep, first, last, **more):
    """`requests` with `cached` = (fewest, most) tokens before the step and `new` in it; each query keeps `keep` pages,
    its first `first` and last `last` among them."""
    return dict(op="select", fmt=fmt, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, requests=requests,
                cached_lo=cached[0], cached_hi=cached[1], new_lo=new[0], new_hi=new[1], keep=keep, first=first, last=last, **more)


def attention_case(fmt, dtype, heads, kv_heads, head_dim, page, requests, cached, new, keep, **more):
    return dict(op="attention", fmt=fmt, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                requests=requests, cached_lo=cached[0], cached_hi=cached[1], new_lo=new[0], new_hi=new[1], keep=keep, **more)


def listed():
    return [
        # a decode step's rows of one layer, straight from the projections in fp32, 64 heads over 8 x 128: latency
        append_case("int4", "fp32", 64, 64, 8, 128, 16, 128, 1, False, 9000, name="append decode int4"),
        # packed prompts with pictures among their tokens: positions of three axes, bandwidth
        append_case("nf4", "bf16", 20011, 28, 4, 128, 32, 128, 3, False, 20011, name="append prompts nf4 3 axes"),
        # half of a 64-wide head turned, in pairs of neighbours, at far positions
        append_case("int4", "fp16", 6007, 32, 8, 64, 64, 32, 1, True, 1000000, name="append prompts int4 64 far"),
        # one user's next token behind 9000: the smallest choice, latency
        select_case("int4", "fp16", 28, 4, 128, 16, 1, (8999, 8999), (1, 1), 64, 1, 2, name="select one 9k"),
        # a serving batch between 8 and 32 thousand tokens, 64 heads over 8
        select_case("int4", "fp16", 64, 8, 128, 64, 32, (8000, 32000), (1, 1), 32, 1, 2, name="select 32 ragged"),
        # one request with a very long context in small pages: 8192 boxes to score and to rank
        select_case("nf4", "bf16", 64, 8, 128, 16, 1, (131070, 131070), (1, 1), 256, 4, 16, name="select one 131k"),
        # a chunk of a long prompt: every token chooses among the pages before it
        select_case("int4", "fp16", 64, 8, 128, 64, 1, (30000, 30000), (1024, 1024), 64, 1, 4, name="select chunk 1024"),
        # requests of every length with drafted tokens, 64-wide heads: some have fewer pages than they may keep
        select_case("nf4", "bf16", 32, 8, 64, 32, 40, (0, 6000), (1, 9), 48, 1, 2, name="select drafts ragged 64"),
        # one user's next token over 16 pages of 64: the smallest attention call
        attention_case("int4", "fp16", 28, 4, 128, 64, 1, (20000, 20000), (1, 1), 16, name="attention one"),
        # a serving batch's decode step, 32 pages of 64 for each of 8 kv heads: cache bandwidth
        attention_case("int4", "fp16", 64, 8, 128, 64, 32, (8000, 32000), (1, 1), 32, name="attention 32 ragged int4"),
        # many requests of every length, 64-wide heads, small pages
        attention_case("nf4", "bf16", 32, 8, 64, 16, 96, (0, 6000), (1, 1), 64, name="attention 96 ragged nf4 64"),
        # a chunk of a prompt, each token with lists of its own
        attention_case("int4", "fp16", 28, 4, 128, 32, 1, (12000, 12000), (300, 300), 32, name="attention chunk int4"),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))

    op = rng.choice(("append", "append", "select", "select", "select", "attention", "attention", "attention"))
    fmt, page = rng.choice(("int4", "nf4")), rng.choice((16, 32, 64))
    kv_heads, head_dim = rng.choice((1, 2, 4, 8, 12)), rng.choice((64, 128, 128))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    if op == "append":
        rotated = head_dim if rng.random() < 0.6 else rng.choice((16, 32, 48, 64))
        axes = rng.choice((1, 1, 2, 3))
        tokens = spread(1, max(1, min(40000, 80_000_000 // (kv_heads * (group + 2) * head_dim))))
        return append_case(fmt, rng.choice(("fp16", "bf16", "fp32")), tokens, group * kv_heads, kv_heads, head_dim, page, rotated, axes,
                           rng.random() < 0.4, spread(100, 1000000))
    while True:
        kind = rng.choice(("decode", "decode", "drafts", "prompt"))
        n = spread(1, 128) if kind != "prompt" else spread(1, 6)
        hi = spread(16, 131072 if n < 4 else 32768)
        cached = (hi, hi) if rng.random() < 0.3 else (rng.randrange(hi + 1), hi)
        new = (1, 1) if kind == "decode" else (rng.choice((0, 2, 3)), rng.randrange(3, 9)) if kind == "drafts" else (rng.randrange(1, 30), spread(30, 1200))
        keep = spread(4, 256)
        if op == "select":
            first, last = rng.randrange(0, max(1, keep // 4)), rng.randrange(1, max(2, keep // 4))
            c = select_case(fmt, rng.choice(("fp16", "bf16")), group * kv_heads, kv_heads, head_dim, page, n, cached, new, keep, first, last)
        else:
            c = attention_case(fmt, rng.choice(("fp16", "bf16")), group * kv_heads, kv_heads, head_dim, page, n, cached, new, keep)
        held, added = lengths(c)
        most, width, total = max(added), max(-(-(a + b) // page) for a, b in zip(held, added)), sum(added)
        if total == 0 or sum(-(-(a + b) // page) * page for a, b in zip(held, added)) * kv_heads * head_dim > 3.0e8:
            continue
        # what the plain forms hold in 32 bits: scores of every page, or every query's own keys
        if op == "select" and n * most * kv_heads * width < 3e7 and work(c)["bytes"] < 6e7:
            return c
        if op == "attention" and total * kv_heads * min(keep, width) * page * head_dim < 1.3e8:
            return c


def lengths(case):
    """The requests' cached and new lengths, spread evenly between their bounds in an order that is not sorted."""
    def between(lo, hi, step):
        return [lo + int((hi - lo + 1) * math.modf((r + 1) * step)[0]) for r in range(case["requests"])]

    return between(case["cached_lo"], case["cached_hi"], 0.6180339887), between(case["new_lo"], case["new_hi"], 0.7548776662)


def code_bytes(case):
    """(bytes of a token's codes, bytes of its scale) in one kv head, keys or values."""
    return case["head_dim"] // 2, 2 if case["fmt"] == "int4" else 4


def out_dtype(case):
    """Rotated queries are of the type that attention takes."""
    return torch.float16 if case["dtype"] == "fp32" else DTYPES[case["dtype"]]


def work(case):
    d, codes, scale = case["head_dim"], *code_bytes(case)
    if case["op"] == "append":
        t, n = case["tokens"], case["tokens"] * case["kv_heads"]
        item = DTYPES[case["dtype"]].itemsize
        # queries in and out, keys and values in, codes and scales out and in again, fp32 values out; positions and slots
        return {"bytes": t * case["heads"] * d * (item + 2) + 2 * n * (d * (item + 4) + 2 * (codes + scale)) + 4 * t * (case["axes"] + 2),
                "flops": 3 * t * (case["heads"] + case["kv_heads"]) * case["rotated"] + 8 * n * d}
    cached, new = lengths(case)
    page, h = case["page"], case["kv_heads"]
    if case["op"] == "select":
        box = 2 * d + 4
        done = scored = pairs = listed_pages = 0
        for c, n in zip(cached, new):
            done += (c + n) // page - c // page
            seen = [(c + i) // page + 1 for i in range(n)]                       # the pages of each query
            some = [max(0, p - case["first"] - case["last"]) if p > case["keep"] else 0 for p in seen]
            pairs += sum(some)
            scored += max(some, default=0)
            listed_pages += sum(min(p, case["keep"]) for p in seen)
        # completed pages' keys in, their boxes out; boxes in, queries in, tables in, lists out
        return {"bytes": h * (done * (page * (codes + scale) + box) + scored * box) + 4 * scored + 2 * sum(new) * case["heads"] * d
                + 4 * h * listed_pages + 4 * sum(new), "flops": 4 * pairs * h * d + 2 * done * page * h * d}
    seen = reads = 0
    for c, n in zip(cached, new):
        visible = [min((c + i) // page, case["keep"] - 1) * page + (c + i) % page + 1 for i in range(n)]
        seen += sum(visible)
        reads += min(sum(visible), c + n)                                         # a page may be in many lists
    return {"bytes": 2 * reads * h * (codes + scale) + 4 * sum(new) * case["heads"] * d + 4 * h * (seen // page + sum(new)),
            "flops": 4 * seen * case["heads"] * d}


# ---- what a program has in hand --------------------------------------------------

def generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = generator(seed)
    state = dict(case=case)
    if case["op"] == "append":
        return prepare_append(case, state, g)
    cached, new = lengths(case)
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
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
    tables = torch.where(column[None, :] < need_t[:, None], order[where.clamp(max=pages - 1)], -1).to(torch.int32)
    state.update(tables=tables, ctx_len=torch.tensor([a + b for a, b in zip(cached, new)], **ints),
                 q_starts=torch.tensor(np.concatenate([[0], np.cumsum(new)]), **ints), max_q=max(new))
    # keys with a few strong columns, values plain; both with tokens of unlike size
    parts, scales = [], []
    for strong in (True, False):
        if not strong and case["op"] == "select":                                 # that reads no values
            parts.append(torch.zeros_like(parts[0]))
            scales.append(torch.zeros_like(scales[0]))
            break
        x = torch.randn((pages, h, page, d), generator=g, device=DEVICE)
        if strong:
            x += torch.randn((pages, h, 1, d), generator=g, device=DEVICE)       # a page's tokens are alike
            x *= 1 + 2 * (torch.rand((1, h, 1, d), generator=g, device=DEVICE) > 0.95)
        x *= torch.exp(0.25 * torch.randn((pages, h, page, 1), generator=g, device=DEVICE))
        amax = x.abs().amax(-1, keepdim=True)
        if case["fmt"] == "int4":
            s = (amax * (1 / 7)).half()
            codes = torch.round(x / s.float()).add_(8).clamp_(0, 15).to(torch.uint8)
        else:
            s = amax
            t = torch.tensor(NF4, device=DEVICE)
            codes = torch.bucketize(x / s, (t[1:] + t[:-1]) / 2, out_int32=True).to(torch.uint8)
        del x
        parts.append((codes[..., 0::2] | codes[..., 1::2] << 4).view(pages, h, -1))
        scales.append(s.view(torch.uint8).view(pages, h, -1))
        del codes
    state["blocks"] = torch.cat(parts + scales, -1).contiguous()
    q = torch.randn((total, case["heads"], d), generator=g, device=DEVICE)
    state["q"] = q.to(DTYPES[case["dtype"]])
    # the step's tokens: their requests, places and slots
    r = torch.repeat_interleave(torch.arange(case["requests"], device=DEVICE), torch.tensor(new, device=DEVICE))
    place = torch.arange(total, device=DEVICE) - state["q_starts"].long()[r] + torch.tensor(cached, device=DEVICE)[r]
    own_page = tables[r, place // page].long()
    slots = own_page * page + place % page
    if case["op"] == "select":
        room = -(-total // 64) * 64                                               # slots are laid out for a step of this many tokens
        state["slots"] = torch.cat([slots, slots.new_full((room - total,), -1)]).to(torch.int32)
        boxes = torch.cat([plain_boxes(case, state["blocks"][at: at + 2048]) for at in range(0, pages, 2048)])
        boxes[own_page[slots % page == page - 1]] = 0                             # those of the pages that this step completes are to come
        state["boxes"] = boxes
        return state
    # lists: a choice of the earlier pages in order, and the query's own page last
    keep, width = case["keep"], max(width, case["keep"])
    mine = place // page
    luck = torch.rand((total, h, width), generator=g, device=DEVICE)
    luck = torch.where(torch.arange(width, device=DEVICE) < mine[:, None, None], luck, -1.0)
    some = luck.topk(min(keep - 1, width), -1) if keep > 1 else None
    seen = torch.minimum(mine, torch.tensor(keep - 1, device=DEVICE))
    blocks = torch.full((total, h, keep), width, device=DEVICE)
    if some is not None:
        blocks[..., : some.indices.shape[-1]] = torch.where(some.values >= 0, some.indices, width)
    blocks = blocks.sort(-1).values
    blocks[torch.arange(total, device=DEVICE)[:, None], torch.arange(h, device=DEVICE), seen[:, None]] = mine[:, None]
    padded = torch.nn.functional.pad(tables, (0, width + 1 - tables.shape[1]), value=-1)
    state["lists"] = padded[r[:, None, None], blocks].contiguous()
    state["seen"] = (seen * page + place % page + 1).to(torch.int32)
    state["out"] = torch.empty_like(state["q"])
    return state


def prepare_append(case, state, g):
    t, n, h, d, page = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    pages = -(-t // page) + 3
    # queries, keys and values are column slices of one fused projection's rows
    rows = torch.randn((t, (n + 2 * h) * d), generator=g, device=DEVICE)
    rows *= torch.exp(0.5 * torch.randn((t, 1), generator=g, device=DEVICE))
    rows = rows.to(DTYPES[case["dtype"]])
    positions = torch.randint(case["far"], (case["axes"], t), generator=g, device=DEVICE, dtype=torch.int32)
    half = case["rotated"] // 2
    pair_axis = [i % case["axes"] for i in range(half)] if case["adjacent"] else [i * case["axes"] // half for i in range(half)]
    state.update(q=rows[:, : n * d].view(t, n, d), k=rows[:, n * d: (n + h) * d].view(t, h, d), v=rows[:, (n + h) * d:].view(t, h, d),
                 positions=positions, inv_freq=[1e6 ** (-i / half) for i in range(half)], pair_axis=pair_axis,
                 slots=torch.randperm(pages * page, generator=g, device=DEVICE)[:t].to(torch.int32),
                 blocks=torch.zeros((pages, h, page * 2 * sum(code_bytes(case))), dtype=torch.uint8, device=DEVICE),
                 q_out=torch.empty((t, n, d), dtype=out_dtype(case), device=DEVICE),
                 k_out=torch.empty((t, h, d), device=DEVICE), v_out=torch.empty((t, h, d), device=DEVICE))
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
    if "lib" not in state:          # the program's imports, its handle of the cache, its table of angles
        at = os.path.join(os.getcwd(), "int4-gemv_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import b4gemv
        state["lib"] = b4gemv
        fmt = b4gemv.KV_INT4 if case["fmt"] == "int4" else b4gemv.KV_NF4
        state["cache"] = b4gemv.KVCache(state["blocks"], fmt, case["page"], case["head_dim"])
        if case["op"] == "append":
            state["rotary"] = b4gemv.Rotary(case["rotated"], inv_freq=state["inv_freq"], axes=state["pair_axis"], adjacent=case["adjacent"],
                                            device=state["blocks"].device)
        if case["op"] == "attention":
            state["chosen"] = b4gemv.KVLists(state["lists"], state["seen"])
    lib, cache = state["lib"], state["cache"]
    if case["op"] == "append":
        q = lib.kv_append_rotary(cache, state["rotary"], state["q"], state["k"], state["v"], state["positions"], state["slots"],
                                 out=state["q_out"])
        k, v = lib.kv_read(cache, state["slots"], state["k_out"], state["v_out"])
        return dict(q=q, k=k, v=v)
    if case["op"] == "select":
        lib.kv_boxes(cache, state["boxes"], state["slots"])
        lists = lib.kv_select(cache, state["boxes"], state["q"], state["tables"], state["ctx_len"], state["q_starts"], state["max_q"],
                              case["keep"], first=case["first"], last=case["last"])
        return dict(pages=lists.pages, seen=lists.seen, boxes=state["boxes"])
    return lib.kv_attention_lists(cache, state["q"], state["chosen"], out=state["out"])


def run_plain(state):
    return dict(append=plain_append, select=plain_select, attention=plain_attention)[state["case"]["op"]](state)


def plain_quantise(case, x):
    """Codes (bytes of two) and scales, as bytes, of x [tokens, kv_heads, head_dim]."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    if case["fmt"] == "int4":
        s = torch.where(amax > 0, amax * (1 / 7), 1.0).half()
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


def plain_angles(state):
    """Cosines and sines [tokens, rotated / 2] in 64 bits: the turns of a position times a frequency, the whole ones left
    out of the product's leading part, which is exact."""
    turns = torch.tensor(state["inv_freq"], dtype=torch.float64, device=DEVICE) / (2 * math.pi)
    lead = torch.round(turns * 2.0 ** 32) / 2.0 ** 32
    at = state["positions"].double()[torch.tensor(state["pair_axis"], device=DEVICE)].T
    whole = at * lead
    part = whole - torch.floor(whole) + at * (turns - lead)
    return torch.cos(2 * math.pi * part), torch.sin(2 * math.pi * part)


def plain_rotate(case, x, c, s):
    r = case["rotated"]
    c, s = c[:, None].to(x.dtype), s[:, None].to(x.dtype)
    if case["adjacent"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., r:]], -1)


def plain_append(state):
    case, blocks, slots = state["case"], state["blocks"], state["slots"].long()
    page = case["page"]
    codes, scale = code_bytes(case)
    c, s = plain_angles(state)
    # keys turn in 64 bits and are rounded to 32 once, so that what lies next to a border between codes has one side
    kb, ks = plain_quantise(case, plain_rotate(case, state["k"].double(), c, s).float())
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
    return dict(q=plain_rotate(case, state["q"].float(), c, s).to(out_dtype(case)),
                k=plain_values(case, blocks[where[0]], blocks[where[2]].view(kind).squeeze(-1).float()),
                v=plain_values(case, blocks[where[1]], blocks[where[3]].view(kind).squeeze(-1).float()))


def plain_boxes(case, blocks):
    """Boxes, as bytes, around the keys of pages [n, kv_heads, block bytes]."""
    codes, _, scales, _ = parts_of(case, blocks)
    k = plain_values(case, codes, scales)
    box = torch.cat([k.amax(-2), k.amin(-2)], -1)
    top = box.abs().amax(-1, keepdim=True)
    s = torch.where(top > 0, top * (1 / 127), 1.0)
    rounded = torch.round(box / s).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return torch.cat([rounded, s.view(torch.uint8), torch.zeros_like(s.view(torch.uint8)).repeat(1, 1, 3)], -1)


def plain_select(state):
    case, q, boxes, tables = state["case"], state["q"], state["boxes"], state["tables"].long()
    ctx, starts, slots = state["ctx_len"].long(), state["q_starts"].long(), state["slots"].long()
    page, h, d, keep, first, last = case["page"], case["kv_heads"], case["head_dim"], case["keep"], case["first"], case["last"]
    b, total, width, most = ctx.shape[0], q.shape[0], tables.shape[1], max(state["max_q"], 1)
    done = slots[slots % page == page - 1] // page
    boxes[done] = plain_boxes(case, state["blocks"][done])
    # the parts of a kv head's queries above and below 0, summed; as int8 in units of their largest
    x = q.double().view(total, h, -1, d)
    x = torch.cat([x.clamp(min=0).sum(2), x.clamp(max=0).sum(2)], -1).float()
    top = x.abs().amax(-1, keepdim=True)
    x = torch.round(x / torch.where(top > 0, top * (1 / 127), 1.0)).clamp(-127, 127)
    # scores of every page of a request, its queries padded to the most: whole numbers below 2^24 times the box's scale
    n = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + torch.arange(most, device=q.device)).clamp(max=total - 1)
    box = boxes[tables.clamp(min=0)]
    codes = box[..., : 2 * d].contiguous().view(torch.int8).float()
    scale = box[..., 2 * d: 2 * d + 4].contiguous().view(torch.float32).squeeze(-1)
    s = torch.einsum("bqhd,bwhd->bqhw", x[at], codes) * scale.transpose(1, 2)[:, None]
    # a query's pages up to its own: the first and the last of them, and the best of the others, ties to the earlier
    place = (ctx - n)[:, None] + torch.arange(most, device=q.device)
    mine = place // page
    column = torch.arange(width, device=q.device)
    fixed = ((column < first) | (column > mine[..., None] - last))[:, :, None]
    s = torch.where(fixed, math.inf, s)
    s = torch.where((column <= mine[..., None])[:, :, None], s, -math.inf)
    if width < keep:
        s = torch.nn.functional.pad(s, (0, keep - width), value=-math.inf)
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = torch.minimum(mine + 1, torch.tensor(keep, device=q.device))
    order = torch.where(torch.arange(keep, device=q.device) < count[:, :, None, None], order, s.shape[-1]).sort(-1).values
    padded = torch.nn.functional.pad(tables, (0, s.shape[-1] + 1 - width), value=-1)
    pages = torch.gather(padded[:, None, None].expand(-1, most, h, -1), -1, order)
    seen = (count - 1) * page + place % page + 1
    token = torch.arange(total, device=q.device)
    r = torch.searchsorted(starts[1:], token, right=True)
    return dict(pages=pages[r, token - starts[r]].int(), seen=seen[r, token - starts[r]].int(), boxes=boxes)


def plain_attention(state):
    case, q, lists, seen = state["case"], state["q"], state["lists"].long(), state["seen"].long()
    total, h, d = q.shape[0], case["kv_heads"], case["head_dim"]
    heads = torch.arange(h, device=q.device)[None, :, None]
    kc, vc, ks, vs = parts_of(case, state["blocks"][lists.clamp(min=0), heads])               # [tokens, h, pages, page, ...]
    k, v = (plain_values(case, c, s).view(total, h, -1, d) for c, s in ((kc, ks), (vc, vs)))
    x = q.float().view(total, h, -1, d)
    s = torch.matmul(x, k.transpose(-1, -2)).mul_(d ** -0.5)
    key = torch.arange(k.shape[2], device=q.device)
    there = (key < seen[:, None, None]) & (lists >= 0).repeat_interleave(case["page"], -1)
    s.masked_fill_(~there[:, :, None], -math.inf)
    p = torch.exp(s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)))
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    return torch.matmul(p, v).view(total, case["heads"], d).to(q.dtype)


# ---- from the definitions, in 64 bits -----------------------------------------------

def exact(case, seed):
    if case["op"] == "select":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return exact_append(case, s)
    q, h, d, page = s["q"].double(), case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // h
    kb, vb, ks, vs = parts_of(case, s["blocks"])
    out = torch.zeros_like(q)
    longest = -(-int(s["seen"].max()) // page)
    rows = max(1, 20_000_000 // (longest * page * d))
    for i in range(h):
        for at in range(0, q.shape[0], rows):
            ids = s["lists"][at: at + rows, i, :longest].long()
            n = ids.shape[0]
            k, v = (exact_values(case, codes[ids, i].reshape(-1, d // 2), scale[ids, i].reshape(-1)).view(n, -1, d)
                    for codes, scale in ((kb, ks), (vb, vs)))
            a = torch.einsum("ngd,nkd->ngk", q[at: at + rows, i * group: (i + 1) * group], k) / math.sqrt(d)
            place = torch.arange(a.shape[-1], device=a.device)
            a = a.masked_fill((place[None] >= s["seen"].long()[at: at + rows, None])[:, None], -math.inf)
            out[at: at + rows, i * group: (i + 1) * group] = torch.einsum("ngk,nkd->ngd", torch.softmax(a, -1), v)
    return out


def exact_values(case, codes, scale):
    low, high = (codes % 16).long(), (codes // 16).long()
    levels = torch.arange(-8, 8, device=codes.device).double() if case["fmt"] == "int4" else \
        torch.tensor(NF4, dtype=torch.float64, device=codes.device)
    values = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64, device=codes.device)
    values[:, 0::2], values[:, 1::2] = levels[low], levels[high]
    return values * scale.double()[:, None]


def exact_append(case, s):
    half = case["rotated"] // 2
    # a position's turns as a whole number of 2^-64 of one, whose carries are the whole turns
    positions = s["positions"].cpu().numpy().astype(np.uint64)
    angle = np.empty((case["tokens"], half))
    for i, (f, axis) in enumerate(zip(s["inv_freq"], s["pair_axis"])):
        step = np.uint64(int(f / (2 * math.pi) * 2 ** 64))
        angle[:, i] = (positions[axis] * step).astype(np.int64) * (math.pi / 2 ** 63)
    turn = torch.from_numpy(np.exp(1j * angle)).to(DEVICE)[:, None]
    parts = {}
    for name in ("q", "k"):
        x = s[name].double()
        pairs = x[..., : 2 * half].unflatten(-1, (half, 2)) if case["adjacent"] else x[..., : 2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.flatten(-2) if case["adjacent"] else z.transpose(-1, -2).flatten(-2)
        parts[name] = torch.cat([z, x[..., 2 * half:]], -1)
    return dict(q=parts["q"], k=exact_rounded(case, parts["k"].float()), v=exact_rounded(case, s["v"].float()))


def exact_rounded(case, x):
    """fp32 x [tokens, kv_heads, head_dim] replaced by the values of its codes: the nearest by the quotient, which is defined in 32 bits."""
    top = x.abs().max(-1, keepdim=True).values
    if case["fmt"] == "int4":
        step = torch.where(top > 0, top * torch.tensor(1 / 7, device=x.device), torch.ones_like(top)).half().double()
        y = (x.double() / step).float().double()
        return torch.clamp(torch.sign(y) * torch.floor(y.abs() + 0.5), -8, 7) * step
    top = torch.where(top > 0, top, torch.ones_like(top)).double()
    levels = torch.tensor(NF4, dtype=torch.float64, device=x.device)
    y = (x.double() / top).float().double().contiguous()
    right = torch.searchsorted(levels, y).clamp(1, 15)
    # the distances too are fp32's
    nearer = (y - levels[right - 1]).float() <= (levels[right] - y).float()
    return levels[right - nearer.long()] * top
