"""Measured cases of the 4-bit paged KV cache: attention over it, the rotary append that
quantises into it, and the page allocator that builds block tables and slot maps from request
lengths.

``run`` computes the plain form (elementary torch operations) where ``own`` is false and calls
``glacier_b200.ops`` where it is true.  ``exact`` computes the definition in 64 bits.

The cache: a page holds 16 positions; the block of one (page, layer, kv head) is ``18 * head_dim``
contiguous bytes

    K codes   [16 positions][4 t][head_dim/32 g] words of 8 codes: dims 32 g + 8 t .. + 7
    V codes   [8 position pairs][head_dim/4 w][2 positions] units of 4 codes: dims 4 w .. 4 w + 3
    K scales  [8 position pairs][head_dim/32 g][2 positions] fp16
    V scales  the same

with codes low nibble first and the value of code u in a group of scale s being s * (u - 7).
A group's scale is the smallest multiple of 2^-21 of at most 7 significant bits with
7 s >= max|x|, at most 7168; a code is 7 + x / s rounded to the nearest integer, ties to even, in
[0, 15].
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 16
LAYERS, LAYER = 2, 1  # the pool holds two layers; the second one is used
MAX_SCALE = 7168.0
THETA = 1e6


def _ops():
    try:
        from glacier_b200 import ops
    except ImportError:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "glacier-engine_b200"))
        from glacier_b200 import ops
    return ops


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

GEOMETRIES = ((14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (16, 2, 128), (4, 4, 128), (6, 3, 64))


def _case(op, geometry, lanes, lo, hi, **more):
    h, k, d = geometry
    return dict(op=op, heads=h, kv_heads=k, head_dim=d, lanes=lanes, lo=lo, hi=hi, **more)


def listed():
    return [
        # one request of the smallest model, a few tokens into its answer: latency
        dict(_case("attend", (14, 2, 64), 1, 40, 40), name="attend one short"),
        # one request of the largest model with a long document in its cache
        dict(_case("attend", (28, 4, 128), 1, 32768, 32768), name="attend one long"),
        # eight requests of very different ages, one slot empty
        dict(_case("attend", (12, 2, 128), 8, 0, 4097), name="attend ragged"),
        # the headline serving batch: 64 lanes with contexts of 256 to 4096
        dict(_case("attend", (28, 4, 128), 64, 256, 4096), name="attend batch"),
        # every lane a step takes, one query head per kv head, odd lengths
        dict(_case("attend", (8, 8, 64), 128, 1, 1999), name="attend many lanes"),
        # the token of one request
        dict(_case("append", (14, 2, 64), 1, 40, 40), name="append one"),
        # the tokens of a full step, or a prompt chunk
        dict(_case("append", (28, 4, 128), 128, 0, 4095), name="append batch"),
        # a decode step's bookkeeping: every request grows by one position
        dict(_case("resize", (28, 4, 128), 64, 256, 4096, grow="one"), name="resize step"),
        # prompts of many requests admitted at once, as one packed batch
        dict(_case("resize", (28, 4, 128), 128, 1, 4096, grow="packed"), name="resize prompts"),
        # the cache's whole part of a decode step, one request
        dict(_case("step", (28, 4, 128), 1, 1000, 1000), name="step one"),
        # the same for a batch
        dict(_case("step", (12, 2, 128), 64, 256, 4095), name="step batch"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "append", "resize", "step"))
    geometry = rng.choice(GEOMETRIES)
    lanes = _log(rng, 1, 128)
    # at most the positions of the largest listed batch in all, so that a case costs no more
    most = min(32768, 64 * 2000 * 4 // (lanes * geometry[1]))
    hi = _log(rng, 1, max(2, most))
    lo = rng.choice((0, 1, hi // 2, hi))
    if op != "resize":
        if op == "append":
            hi, lo = min(hi, 8191), min(lo, 8191)
        return _case(op, geometry, lanes, lo, hi)
    # in one of three the free pages do not last for every request
    hi, lo = min(hi, 4096), min(lo, 4096)
    return _case(op, geometry, lanes, lo, hi, grow=rng.choice(("one", "packed")), short=rng.random() < 0.33)


def _lengths(case):
    """Contexts of the lanes: from the case alone, so that its work is known without its inputs."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k != "name"))
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["lanes"])]
    if case["lo"] < case["hi"]:
        lens[-1] = case["hi"]
    return lens


def _pages(n):
    return -(-n // PAGE)


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _block_bytes(hd):
    return 18 * hd


def _random_pool(g, pages, hkv, hd):
    """A pool of quantised pages: codes of a normal distribution, scales of varied size."""
    dev = "cuda"
    blk = _block_bytes(hd)
    pool = torch.empty((pages, LAYERS, hkv, blk), dtype=torch.uint8, device=dev)
    n = torch.randn(pool.shape, generator=g, dtype=torch.float16, device=dev)
    lo = (n * 2.6).round_().clamp_(-7, 8).add_(7).to(torch.uint8)
    n = torch.randn(pool.shape, generator=g, dtype=torch.float16, device=dev)
    hi = (n * 2.6).round_().clamp_(-7, 8).add_(7).to(torch.uint8)
    torch.bitwise_or(lo, hi << 4, out=pool)
    del n, lo, hi
    s = torch.rand((pages, LAYERS, hkv, hd), generator=g, dtype=torch.float32, device=dev).mul_(0.4).add_(0.15)
    # 7 significant bits: 6 stored mantissa bits of the fp16 number
    s = (s.half().view(torch.int16) & -16)
    pool[..., 16 * hd:] = s.view(torch.uint8)
    return pool


def _rope(positions, hd):
    i = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * THETA ** (-2.0 * i / hd)
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h, hkv, hd, lanes, op = case["heads"], case["kv_heads"], case["head_dim"], case["lanes"], case["op"]
    lens = _lengths(case)
    st = dict(op=op, h=h, hkv=hkv, hd=hd, lanes=lanes)
    dev = torch.device("cuda")
    i32 = dict(dtype=torch.int32, device=dev)
    lens_t = torch.tensor(lens, **i32)
    if op == "resize":
        old = [0] * lanes if case["grow"] == "packed" else lens
        new = lens if case["grow"] == "packed" else [n + 1 for n in lens]
    elif op == "step":
        old, new = lens, [n + 1 for n in lens]
    else:
        old = new = lens
    max_pages = max(1, max(_pages(n) for n in new) + (1 if op == "append" else 0))
    held = [_pages(n) for n in old]
    # the pool holds every lane's final pages and a few more, placed at random
    total = sum(_pages(n) for n in new) + lanes + 3
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.full((lanes, max_pages), -1, **i32)
    take = torch.tensor(held, **i32)
    mask = torch.arange(max_pages, device=dev)[None] < take[:, None]
    table[mask] = perm[:sum(held)]
    st.update(table=table, max_pages=max_pages)
    if op in ("resize", "step"):
        one = op == "step" or case["grow"] == "one"
        rows = lanes if one else max(1, sum(new))
        free = perm[sum(held):].flip(0).contiguous()
        if case.get("short"):
            free = free[:max(1, free.numel() // 3)]
        stack = torch.full((total,), -1, **i32)
        stack[:free.numel()] = free
        st.update(lens=torch.tensor(old, **i32), targets=torch.tensor(new, **i32), back=torch.tensor(old, **i32),
                  free=stack, count=torch.tensor([free.numel()], **i32), rows=rows, stride=1 if one else 0,
                  positions=torch.empty(rows, **i32), row_lanes=torch.empty(rows, **i32),
                  slots=torch.empty(rows, dtype=torch.int64, device=dev), offsets=torch.empty(lanes + 1, **i32),
                  status=torch.empty(lanes, **i32), status_back=torch.empty(lanes, **i32))
    if op == "resize":
        return st
    st["pool"] = _random_pool(g, total, hkv, hd).view(total, -1)
    st["q"] = torch.randn((lanes, h * hd), generator=g, device=dev)
    if op in ("append", "step"):
        st["qkv"] = torch.randn((lanes, (h + 2 * hkv) * hd), generator=g, device=dev) * 1.5
        st["bias"] = torch.randn((h + 2 * hkv) * hd, generator=g, device=dev) * 0.5
        st["cos"], st["sin"] = _rope(max_pages * PAGE, hd)
        st["q"] = torch.empty((lanes, h * hd), device=dev)
    if op == "append":
        # each row goes to its lane's next position; one row of a larger batch is padding
        last = perm[sum(held):sum(held) + lanes].long()
        page = torch.where(lens_t % PAGE == 0, last, table.gather(1, (lens_t.long() // PAGE)[:, None])[:, 0].long())
        st["slots"] = page * PAGE + lens_t % PAGE
        st["positions"] = lens_t
        if lanes > 4:
            st["slots"][2] = -1
    if op == "attend":
        st["ctx"] = lens_t
    if op in ("attend", "step"):
        st["out"] = torch.empty((lanes, h * hd), device=dev)
    return st


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------

def _values(blocks, hd):
    """K and V values [n, 16, hd] of blocks [n, 18 hd] of bytes."""
    n, ng = blocks.shape[0], hd // 32
    half = hd // 2
    k = blocks[:, :16 * half].reshape(n, 16, 4, ng, 4)
    k = torch.stack((k & 15, k >> 4), -1).permute(0, 1, 3, 2, 4, 5).reshape(n, 16, ng, 32)
    v = blocks[:, 16 * half:32 * half].reshape(n, 8, hd // 4, 2, 2)
    v = torch.stack((v & 15, v >> 4), -1).permute(0, 1, 3, 2, 4, 5).reshape(n, 16, ng, 32)
    s = blocks[:, 16 * hd:].contiguous().view(torch.float16).reshape(n, 2, 8, ng, 2).permute(0, 1, 2, 4, 3)
    s = s.reshape(n, 2, 16, ng, 1).float()
    return ((k.float() - 7) * s[:, 0]).reshape(n, 16, hd), ((v.float() - 7) * s[:, 1]).reshape(n, 16, hd)


def _plain_attend(st, q, ctx):
    h, hkv, hd, lanes = st["h"], st["hkv"], st["hd"], st["lanes"]
    pool = st["pool"].view(-1, LAYERS, hkv, _block_bytes(hd))[:, LAYER]
    n = st["max_pages"] * PAGE
    blocks = pool[st["table"].long().clamp(min=0)]  # [lanes, pages, hkv, bytes]
    k, v = _values(blocks.reshape(-1, _block_bytes(hd)), hd)
    k = k.view(lanes, -1, hkv, PAGE, hd).transpose(1, 2).reshape(lanes, hkv, n, hd)
    v = v.view(lanes, -1, hkv, PAGE, hd).transpose(1, 2).reshape(lanes, hkv, n, hd)
    s = torch.matmul(q.view(lanes, hkv, h // hkv, hd), k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    s = s.masked_fill((torch.arange(n, device=q.device)[None] >= ctx[:, None])[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(lanes, h * hd)


def _plain_quantise(x):
    """(scales [.., hd/32] fp16, codes [.., hd] uint8) of rows [.., hd], in 64 bits."""
    x = x.double().reshape(*x.shape[:-1], -1, 32)
    t = x.abs().amax(-1) / 7
    unit = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -40)))) / 64
    # a logarithm next to a power of two may be off by one
    unit = torch.where(t >= unit * 128, unit * 2, torch.where(t < unit * 64, unit / 2, unit)).clamp(min=2.0 ** -21)
    s = (torch.ceil(t / unit) * unit).clamp(max=MAX_SCALE)
    u = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[..., None]).clamp(-7, 8) + 7
    return s.half(), u.to(torch.uint8).flatten(-2)


def _plain_append(st, pos, slots):
    """Rotates, quantises and writes; returns (q, K rows, V rows) as the values that are held."""
    h, hkv, hd = st["h"], st["hkv"], st["hd"]
    x = (st["qkv"] + st["bias"]).view(-1, h + 2 * hkv, hd)
    c, s = st["cos"][pos.long()][:, None], st["sin"][pos.long()][:, None]
    a, b = x[:, :h + hkv, :hd // 2], x[:, :h + hkv, hd // 2:]
    r = torch.cat((a * c - b * s, a * s + b * c), -1)
    q, k, v = r[:, :h], r[:, h:], x[:, h + hkv:]
    ng = hd // 32
    (ks, ku), (vs, vu) = _plain_quantise(k), _plain_quantise(v)
    # K: words (t, g) of 8 codes; V: units of 4 codes, interleaved with the pair's other position
    kb = ku.view(-1, hkv, ng, 4, 4, 2).permute(0, 1, 3, 2, 4, 5)
    kb = (kb[..., 0] | kb[..., 1] << 4).reshape(-1, hkv, hd // 2)
    vb = vu.view(-1, hkv, hd // 4, 2, 2)
    vb = vb[..., 0] | vb[..., 1] << 4
    keep = slots >= 0
    sl = slots[keep]
    page, row = sl // PAGE, sl % PAGE
    pool = st["pool"].view(-1, LAYERS, hkv, _block_bytes(hd))
    pool[:, LAYER, :, :8 * hd].view(-1, hkv, 16, hd // 2)[page, :, row] = kb[keep]
    pool[:, LAYER, :, 8 * hd:16 * hd].view(-1, hkv, 8, hd // 4, 2, 2)[page, :, row // 2, :, row % 2] = vb[keep]
    for_scales = pool[:, LAYER, :, 16 * hd:].view(-1, hkv, 2, 8, ng, 2, 2)
    both = torch.stack((ks, vs), 2)[keep].view(torch.uint8).view(-1, hkv, 2, ng, 2)
    for_scales[page, :, :, row // 2, :, row % 2] = both
    live = keep.view(-1, 1, 1, 1)
    q = torch.where(live[..., 0], q, torch.zeros_like(q))

    def held(u, s):
        w = (u.view(-1, hkv, ng, 32).float() - 7) * s.float()[..., None]
        return torch.where(live, w, torch.zeros_like(w)).reshape(-1, hkv * hd)
    return q.reshape(-1, h * hd), held(ku, ks), held(vu, vs)


def _plain_resize(st):
    """New tables and the row arrays of growing from lens to targets; the growth is taken back."""
    old, new, table, rows, stride = st["lens"].long(), st["targets"].long(), st["table"], st["rows"], st["stride"]
    lanes, max_pages = table.shape
    dev = old.device
    have, want = (old + PAGE - 1) // PAGE, (new + PAGE - 1) // PAGE
    need, add = (want - have).clamp(min=0), (new - old).clamp(min=0)
    valid = (new >= 0) & (new <= max_pages * PAGE) & ((add <= stride) if stride else (add >= 0))
    need, add = need * valid, add * valid
    ok = valid & ((need == 0) | (need.cumsum(0) <= st["count"])) & ((add == 0) | (add.cumsum(0) <= rows))
    status = torch.where(valid, torch.where(ok, 0, -3), -1).to(torch.int32)
    add, first = add * ok, need.cumsum(0) - need
    j = torch.arange(max_pages, device=dev)[None]
    fresh = (j >= have[:, None]) & (j < want[:, None]) & ok[:, None]
    at = (st["count"].long() - 1 - (first[:, None] + j - have[:, None])).clamp(0, st["free"].numel() - 1)
    table = torch.where(fresh, st["free"][at], table)
    ends = add.cumsum(0)
    offsets = torch.cat((torch.zeros_like(ends[:1]), ends))
    r = torch.arange(rows, device=dev)
    if stride:
        lane, i = r // stride, r % stride
        offsets = torch.arange(lanes + 1, device=dev) * stride
    else:
        lane = torch.searchsorted(ends, r, right=True).clamp(max=lanes - 1)
        i = r - offsets[lane]
    live = i < add[lane]
    pos = old[lane] + i
    slot = table[lane, (pos // PAGE).clamp(0, max_pages - 1)].long() * PAGE + pos % PAGE
    none = torch.full_like(slot, -1)
    return dict(table=table, positions=torch.where(live, pos, none).to(torch.int32),
                row_lanes=torch.where(live, lane, none).to(torch.int32), slots=torch.where(live, slot, none),
                offsets=offsets.to(torch.int32), status=status)


def run(st):
    op = st["op"]
    if own:
        return _own(st)
    if op == "attend":
        return _plain_attend(st, st["q"], st["ctx"])
    if op == "append":
        q, k, v = _plain_append(st, st["positions"], st["slots"])
        return dict(q=q, k=k, v=v)
    got = _plain_resize(st)
    if op == "resize":
        return got
    st["table"].copy_(got["table"])
    q, _, _ = _plain_append(st, got["positions"], got["slots"])
    return dict(out=_plain_attend(st, q, st["targets"]), slots=got["slots"])


def _attend(ops, st, q, ctx):
    if "workspace" not in st:  # kept by a program that decodes, as its output buffer
        st["workspace"] = ops.paged_attention_q4_workspace(st["h"], st["hkv"], st["hd"])
    return ops.paged_attention_q4(q, st["pool"], st["table"], ctx, LAYERS, LAYER, st["h"], st["hkv"], st["hd"],
                                  out=st["out"], workspace=st["workspace"])


def _own(st):
    ops = _ops()
    op, h, hkv, hd = st["op"], st["h"], st["hkv"], st["hd"]
    if op == "attend":
        return _attend(ops, st, st["q"], st["ctx"])
    if op == "append":
        q = ops.qkv_rope_append_q4(st["qkv"], st["bias"], st["cos"], st["sin"], st["positions"], st["slots"], h, hkv,
                                   hd, st["pool"], LAYERS, LAYER, q_out=st["q"])
        k, v = ops.kv_q4_read(st["pool"], st["slots"], LAYERS, LAYER, hkv, hd)
        return dict(q=q, k=k, v=v)
    # every request grows, and after the pass goes back to where it was
    ops.kv_resize(st["lens"], st["targets"], st["table"], st["free"], st["count"], st["status"],
                  positions=st["positions"], row_lanes=st["row_lanes"], slots=st["slots"], row_offsets=st["offsets"],
                  row_stride=st["stride"])
    out = None
    if op == "step":
        q = ops.qkv_rope_append_q4(st["qkv"], st["bias"], st["cos"], st["sin"], st["positions"], st["slots"], h, hkv,
                                   hd, st["pool"], LAYERS, LAYER, q_out=st["q"])
        out = _attend(ops, st, q, st["lens"])
    ops.kv_resize(st["lens"], st["back"], st["table"], st["free"], st["count"], st["status_back"])
    if op == "step":
        return dict(out=out, slots=st["slots"])
    return dict(table=st["table"], positions=st["positions"], row_lanes=st["row_lanes"], slots=st["slots"],
                offsets=st["offsets"], status=st["status"])


# ---------------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------------

def work(case):
    h, hkv, hd, lanes, op = case["heads"], case["kv_heads"], case["head_dim"], case["lanes"], case["op"]
    lens = _lengths(case)
    nbytes = flops = 0
    if op == "step":
        lens = [n + 1 for n in lens]
    if op in ("attend", "step"):
        nbytes += sum(lens) * hkv * _block_bytes(hd) // PAGE + sum(_pages(n) for n in lens) * 4 + lanes * (8 * h * hd + 4)
        flops += 4 * h * hd * sum(lens)
    if op in ("append", "step"):
        row = (h + 2 * hkv) * hd * 4 + h * hd * 4 + hkv * _block_bytes(hd) // PAGE + hd * 4 + 12
        nbytes += lanes * row + (h + 2 * hkv) * hd * 4
        flops += lanes * (3 * (h + hkv) * hd + 4 * hkv * hd)
    if op == "append":
        nbytes += lanes * (hkv * _block_bytes(hd) // PAGE + 8 * hkv * hd)  # the rows read back
    if op in ("resize", "step"):
        packed = op == "resize" and case["grow"] == "packed"
        rows = sum(lens) if packed else lanes
        fresh = sum(_pages(n) for n in lens) if packed else 0
        nbytes += rows * 16 + fresh * 16 + lanes * 36
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------

def _cells(pool, page, row, head, hkv, hd, kind):
    """float64 values [n, hd] of positions (page, row) of one kv head, cell by cell from the layout."""
    dev = pool.device
    d = torch.arange(hd, device=dev)
    flat = pool.reshape(-1)
    base = ((page.long() * LAYERS + LAYER) * hkv + head) * (18 * hd)
    base, row = base[:, None], row.long()[:, None]
    if kind == 0:
        byte = row * (hd // 2) + ((d % 32) // 8 * (hd // 32) + d // 32) * 4 + d % 8 // 2
    else:
        byte = 8 * hd + row // 2 * hd + d // 4 * 4 + row % 2 * 2 + d % 4 // 2
    u = (flat[base + byte].to(torch.int64) >> (d % 2 * 4)) & 15
    at = 16 * hd + kind * hd + 2 * (row // 2 * (hd // 16) + d // 32 * 2 + row % 2)
    bits = flat[base + at].to(torch.int64) | flat[base + at + 1].to(torch.int64) << 8
    exponent, mantissa = bits >> 10 & 31, bits & 1023
    s = torch.where(exponent > 0, (1024 + mantissa) * 2.0 ** (exponent - 25).double(), mantissa * 2.0 ** -24)
    return (u - 7) * s


def _exact_attend(st, q, lens):
    h, hkv, hd = st["h"], st["hkv"], st["hd"]
    out = torch.zeros((st["lanes"], h, hd), dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        p = torch.arange(n, device=q.device)
        page, row = st["table"][b].long()[p // PAGE], p % PAGE
        for j in range(hkv):
            heads = slice(j * (h // hkv), (j + 1) * (h // hkv))
            k, v = (_cells(st["pool"], page, row, j, hkv, hd, kind) for kind in (0, 1))
            out[b, heads] = torch.softmax(q[b].double().view(h, hd)[heads] @ k.T / math.sqrt(hd), -1) @ v
    return out.reshape(st["lanes"], -1)


def _f32(x):
    return x.float().double()


def _exact_rows(st, pos):
    """The float32 rows that go into the cache, each rounding of the definition made from 64 bits."""
    h, hkv, hd = st["h"], st["hkv"], st["hd"]
    x = _f32(st["qkv"].double() + st["bias"].double()).view(-1, h + 2 * hkv, hd)
    c, s = st["cos"].double()[pos.long()][:, None], st["sin"].double()[pos.long()][:, None]
    a, b = x[:, :h + hkv].chunk(2, -1)
    lo, hi = (a * c, b * s), (a * s, b * c)
    k = torch.cat((_f32(_f32(lo[0]) - _f32(lo[1])), _f32(_f32(hi[0]) + _f32(hi[1]))), -1)[:, h:]
    q = torch.cat((lo[0] - lo[1], hi[0] + hi[1]), -1)[:, :h]
    return q, k, x[:, h + hkv:]


def _exact_held(x):
    """The values that a row is held as: scale by search over the 7-bit mantissas."""
    n, hkv, hd = x.shape
    g = x.reshape(n, hkv, hd // 32, 32)
    top = g.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top / 7)  # in [1/2, 1)
    step = torch.ldexp(torch.ones_like(mantissa), (exponent - 7).clamp(min=-21))
    s = torch.floor(top / 7 / step) * step
    s = torch.where(7 * s < top, s + step, s).clamp(max=MAX_SCALE)
    t = g / torch.where(s > 0, s, torch.ones_like(s))
    low = torch.floor(t)
    up = (t - low > 0.5) | ((t - low == 0.5) & (low % 2 != 0))
    return ((low + up).clamp(-7, 8) * s).reshape(n, hkv * hd)


def exact(case, seed):
    st = prepare(case, seed)
    op, h, hd = st["op"], st["h"], st["hd"]
    if op == "attend":
        return _exact_attend(st, st["q"], _lengths(case))
    if op == "append":
        q, k, v = _exact_rows(st, st["positions"])
        live = (st["slots"] >= 0).double()[:, None]
        return dict(q=q.reshape(-1, h * hd) * live, k=_exact_held(k) * live, v=_exact_held(v) * live)
    if op == "resize":
        return None
    # a step: place the new rows by hand, then attend over the held values
    hkv, lens = st["hkv"], _lengths(case)
    pos = torch.tensor(lens, device="cuda")
    q, k, v = _exact_rows(st, pos)
    kv = [_exact_held(k).view(-1, hkv, hd), _exact_held(v).view(-1, hkv, hd)]
    out = torch.zeros((len(lens), h, hd), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        p = torch.arange(n, device="cuda")
        page, row = st["table"][b].long()[p // PAGE], p % PAGE
        for j in range(hkv):
            heads = slice(j * (h // hkv), (j + 1) * (h // hkv))
            ks, vs = (torch.cat((_cells(st["pool"], page, row, j, hkv, hd, i), kv[i][b, j][None])) for i in (0, 1))
            out[b, heads] = torch.softmax(q[b].view(h, hd)[heads] @ ks.T / math.sqrt(hd), -1) @ vs
    return dict(out=out.reshape(len(lens), -1), slots=None)
