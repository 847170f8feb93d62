"""The 4-bit paged KV cache (kv_resize, qkv_rope_append_q4, kv_q4_read, paged_attention_q4)
against plain 64-bit implementations, at the sizes and masks where it can go wrong.

Tolerances.  Codes, scales and the page bookkeeping are exact: no tolerance.  The rotated q is a
product sum of two float32 roundings each plus the sum's: at most 3 half steps of 2^-24 relative to
|x0| + |x1|.  An attention output is a weighted mean of held values, which are exact.  A score of
n products carries at most n + 16 half steps of 2^-24 of sum |q k|: its additions (a tensor core that
cuts instead of rounding takes two for each of fewer, longer ones), 4 for q as the sum of two fp16 numbers
(2^-22), the rest for scale, maximum and exponent.  A score's error is its weight's relative error, and
a weighted mean moves by at most twice that times max |v|.  The sums over positions are cut into
warps and tiles of 16 or more, so 2 * 32 half steps cover them at the lengths below:

    tol = 2^-24 * (2 * (n + 16) * max_p sum |q k| / sqrt(n) + 64) * max |v|,   n = head_dim
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu
MAX_SCALE = 7168.0
EINVAL, ENOMEM = -1, -3


# ---- the format, in numpy ----

def scale_of(top):
    """Smallest multiple of 2^-21 of at most 7 significant bits with 7 s >= top, at most 7168."""
    if top == 0:
        return 0.0
    t = top / 7
    step = max(2.0 ** (math.floor(math.log2(t)) - 6), 2.0 ** -21)
    s = math.floor(t / step) * step
    while 7 * s < top:
        s += step
    return min(s, MAX_SCALE)


def quantise(row):
    """(scales [n/32], codes [n]) of one float32 row."""
    g = np.asarray(row, np.float64).reshape(-1, 32)
    scales, codes = [], []
    for x in g:
        if not np.isfinite(x).all():
            scales.append(np.nan)
            codes.append(np.full(32, 7, np.int64))
            continue
        s = scale_of(np.abs(x).max())
        scales.append(s)
        codes.append(np.clip(np.rint(x / s), -7, 8).astype(np.int64) + 7 if s else np.full(32, 7, np.int64))
    return np.array(scales), np.concatenate(codes)


def held(row):
    s, u = quantise(row)
    return np.repeat(s, 32) * (u - 7)


class Pool:
    """A host copy of a pool and its cells, read by the documented byte layout."""

    def __init__(self, data, layers, hkv, hd):
        self.data = np.ascontiguousarray(data).reshape(-1)
        self.layers, self.hkv, self.hd = layers, hkv, hd

    def block(self, page, layer, head):
        n = 18 * self.hd
        o = ((page * self.layers + layer) * self.hkv + head) * n
        return self.data[o:o + n]

    def row(self, page, r, layer, head, kind):
        hd, blk = self.hd, self.block(page, layer, head)
        out = np.empty(hd)
        for d in range(hd):
            if kind == 0:
                byte = r * hd // 2 + ((d % 32 // 8) * (hd // 32) + d // 32) * 4 + d % 8 // 2
            else:
                byte = 8 * hd + r // 2 * hd + d // 4 * 4 + r % 2 * 2 + d % 4 // 2
            at = (16 + kind) * hd + 2 * (r // 2 * 2 * (hd // 32) + d // 32 * 2 + r % 2)
            s = np.frombuffer(blk[at:at + 2].tobytes(), np.float16)[0]
            out[d] = float(s) * (int(blk[byte] >> (d % 2 * 4)) % 16 - 7)
        return out

    def rows(self, table, ctx, layer, head, kind):
        return np.stack([self.row(table[p // 16], p % 16, layer, head, kind) for p in range(ctx)])


def attend64(q, k, v):
    """softmax(q k^T / sqrt(n)) v in 64 bits."""
    s = q.astype(np.float64) @ k.T / math.sqrt(q.shape[1])
    e = np.exp(s - s.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True) @ v


def tolerance(q, k, v):
    n = q.shape[1]
    size = (np.abs(q.astype(np.float64)) @ np.abs(k).T).max() / math.sqrt(n)
    return 2.0 ** -24 * (2 * (n + 16) * size + 64) * np.abs(v).max()


def random_pool(rng, pages, layers, hkv, hd, spread=0.3):
    """Random codes; scales of 7 significant bits."""
    blk = np.empty((pages * layers * hkv, 18 * hd), np.uint8)
    blk[:, :16 * hd] = rng.integers(0, 256, (len(blk), 16 * hd))
    s = (rng.random((len(blk), hd)) * spread + 0.05).astype(np.float16)
    blk[:, 16 * hd:] = (s.view(np.int16) & -16).view(np.uint8).reshape(len(blk), -1)
    return blk.reshape(pages, -1)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def status_word():
    from glacier_b200._lib import lib
    return lib().glacier_cuda_device_status(1)


# ---- refusals (no GPU: every check comes before a launch) ----

def capi(name, *args):
    from glacier_b200._lib import lib
    return getattr(lib(), name)(*args)


def attend_args(**over):
    a = dict(q=4096, pool=4096, num_pages=8, num_layers=2, tables=4096, max_pages=4, ctx=4096, lanes=2, layer=1,
             h=8, hkv=2, hd=64, out=4096, ws=4096, ws_floats=1 << 24)
    a.update(over)
    return tuple(a.values()) + (None,)


@pytest.mark.parametrize("over", [
    dict(hd=96), dict(hd=32), dict(h=7), dict(h=18), dict(hkv=0), dict(layer=2), dict(num_pages=0), dict(lanes=0),
    dict(lanes=1025), dict(max_pages=0), dict(pool=4104), dict(q=4100), dict(out=4100), dict(ws=4100),
    dict(ws_floats=16), dict(q=None), dict(tables=None), dict(ctx=None), dict(out=None), dict(ws=None)])
def test_attention_refusals(over):
    assert capi("glacier_cuda_paged_attention_q4", *attend_args(**over)) == EINVAL


@pytest.mark.parametrize("over", [
    dict(hd=96), dict(h=7), dict(h=24), dict(hkv=0), dict(layer=2), dict(num_pages=0), dict(pool=4104), dict(ld=10),
    dict(ldq=10), dict(positions=0), dict(qkv=None), dict(cos=None), dict(pos=None), dict(slots=None), dict(q=None)])
def test_append_refusals(over):
    a = dict(qkv=4096, ld=768, bias=None, cos=4096, sin=4096, positions=64, pos=4096, slots=4096, batch=2, h=8, hkv=2,
             hd=64, q=4096, ldq=512, pool=4096, num_pages=8, num_layers=2, layer=1)
    a.update(over)
    assert capi("glacier_cuda_qkv_rope_append_q4", *a.values(), None) == EINVAL


@pytest.mark.parametrize("over", [dict(hd=80), dict(layer=2), dict(slots=None), dict(k=4100), dict(v=None)])
def test_read_refusals(over):
    a = dict(pool=4096, num_pages=8, num_layers=2, layer=1, hkv=2, hd=64, slots=4096, rows=3, k=4096, v=4096)
    a.update(over)
    assert capi("glacier_cuda_kv_q4_read_f32", *a.values(), None) == EINVAL


@pytest.mark.parametrize("over", [
    dict(lanes=0), dict(lanes=1025), dict(max_pages=0), dict(capacity=0), dict(lens=None), dict(targets=None),
    dict(targets=4096), dict(tables=None), dict(free=None), dict(count=None), dict(status=None), dict(positions=None),
    dict(slots=None), dict(row_lanes=None), dict(stride=2, rows=7), dict(rows=0)])
def test_resize_refusals(over):
    a = dict(lens=4096, targets=8192, lanes=4, tables=4096, max_pages=4, free=4096, capacity=16, count=4096,
             status=4096, stride=0, rows=8, positions=4096, row_lanes=4096, slots=4096, offsets=None)
    a.update(over)
    assert capi("glacier_cuda_kv_resize", *a.values(), None) == EINVAL


def test_page_bytes_and_workspace():
    assert capi("glacier_cuda_kv_q4_page_bytes", 28, 4, 128) == 28 * 4 * 2304
    assert capi("glacier_cuda_kv_q4_page_bytes", 1, 2, 64) == 2 * 1152
    assert capi("glacier_cuda_paged_attention_q4_workspace", 28, 4, 128) > 0
    assert capi("glacier_cuda_paged_attention_q4_workspace", 28, 0, 128) == 0


def test_wrappers_refuse_other_types_layouts_and_devices():
    from glacier_b200 import ops
    from glacier_b200._lib import GlacierCudaError
    z = lambda *s, d=torch.float32: torch.zeros(s, dtype=d)  # noqa: E731
    i = torch.int32
    pages = z(4, ops.kv_q4_page_bytes(2, 2, 64), d=torch.uint8)
    good = dict(q=z(2, 512), pages=pages, block_tables=z(2, 3, d=i), ctx_lens=z(2, d=i))
    for bad in (dict(q=z(2, 512, d=torch.float16)), dict(q=z(2, 500)), dict(q=z(512, 2).t()),
                dict(pages=pages[:, :-2]), dict(pages=z(4, 7, d=torch.uint8)), dict(block_tables=z(3, 3, d=i)),
                dict(block_tables=z(2, 6, d=i)[:, ::2]), dict(ctx_lens=z(2, d=torch.int64)), {}):  # {}: on the CPU
        with pytest.raises(GlacierCudaError):
            ops.paged_attention_q4(**{**good, **bad}, num_layers=2, layer=0, num_heads=8, num_kv_heads=2, head_dim=64)
    with pytest.raises(GlacierCudaError):
        ops.kv_resize(z(2, d=i), z(2, d=i), z(2, 3, d=i), z(8, d=i), z(1, d=i), z(2, d=i), positions=z(4, d=i))
    with pytest.raises(GlacierCudaError):
        ops.qkv_rope_append_q4(z(2, 700), None, z(16, 32), z(16, 32), z(2, d=i), z(2, d=torch.int64), 8, 2, 64, pages,
                               2, 0)
    with pytest.raises(GlacierCudaError):
        ops.kv_q4_read(pages, z(2, d=i), 2, 0, 2, 64)


# ---- append and read ----

EDGE_ROWS = [
    np.zeros(32), np.full(32, 1e-30), np.full(32, 2.0 ** -21 * 7), np.linspace(-1, 1, 32), np.full(32, 7.0),
    np.arange(32) - 15.5, np.full(32, 5e4), np.full(32, 50176.0), np.linspace(-1e6, 1e6, 32), np.full(32, 3.4e38),
    np.r_[np.full(31, 0.5), 7.0], np.r_[np.full(31, -2.5), 7.0], np.r_[np.full(31, 3.5), -7.0],
    np.r_[np.full(31, 1.0 + 2.0 ** -23), 7.0 + 2.0 ** -21], np.r_[np.zeros(31), np.inf], np.r_[np.nan, np.ones(31)],
    np.r_[np.full(31, 3e-6), 1e-5], np.full(32, -1e-7)]


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_append_holds_what_the_format_says_at_its_edges(hd):
    """No rotation (position 0), no bias: K and V rows of edge values are held exactly as defined."""
    from glacier_b200 import ops
    hkv, h, layers = 2, 2, 2
    n = len(EDGE_ROWS)
    x = np.zeros((n, (h + 2 * hkv) * hd), np.float32)
    for i in range(n):
        groups = [EDGE_ROWS[(i + j) % n] for j in range(2 * hkv * hd // 32)]
        x[i, h * hd:] = np.concatenate(groups).astype(np.float32)
    cos, sin = np.ones((4, hd // 2), np.float32), np.zeros((4, hd // 2), np.float32)
    # a rotation by 0 of a NaN or an infinity multiplies it by sin 0: NaN in the partner's group too
    pages = dev(np.full((3, ops.kv_q4_page_bytes(layers, hkv, hd)), 0xA5, np.uint8))
    slots = dev(np.arange(n, dtype=np.int64) + 5)
    ops.qkv_rope_append_q4(dev(x), None, dev(cos), dev(sin), dev(np.zeros(n, np.int32)), slots, h, hkv, hd, pages,
                           layers, 1)
    k, v = (host(t).reshape(n, hkv, hd) for t in ops.kv_q4_read(pages, slots, layers, 1, hkv, hd))
    pool = Pool(host(pages), layers, hkv, hd)
    for i in range(n):
        for j in range(hkv):
            row = x[i, (h + j) * hd:(h + j + 1) * hd]
            a, b = row[:hd // 2], row[hd // 2:]
            with np.errstate(invalid="ignore"):
                rot = np.concatenate((a * 1 - b * np.float32(0), a * np.float32(0) + b * 1))
            ref_k, ref_v = held(rot), held(x[i, (h + hkv + j) * hd:(h + hkv + j + 1) * hd])
            np.testing.assert_array_equal(k[i, j], ref_k)
            np.testing.assert_array_equal(v[i, j], ref_v)
            slot = i + 5
            np.testing.assert_array_equal(pool.row(slot // 16, slot % 16, 1, j, 0), ref_k)
            np.testing.assert_array_equal(pool.row(slot // 16, slot % 16, 1, j, 1), ref_v)
    # the other layer, and positions that no slot names, are as they were
    data = host(pages).reshape(3, layers, -1)
    assert (data[:, 0] == 0xA5).all()
    for slot in (4, 5 + n):
        for j in range(hkv):
            blk = pool.block(slot // 16, 1, j)
            r = slot % 16
            assert (blk[r * hd // 2:(r + 1) * hd // 2] == 0xA5).all()
            assert (blk[8 * hd + r // 2 * hd:][:hd].reshape(-1, 2, 2)[:, r % 2] == 0xA5).all()
    assert status_word() == 0


@gpu
@pytest.mark.parametrize("h,hkv,hd,batch", [(14, 2, 64, 1), (28, 4, 128, 5), (8, 8, 64, 3), (3, 3, 128, 33),
                                            (16, 2, 128, 128), (5, 1, 64, 2)])
@pytest.mark.parametrize("odd", [False, True])  # odd: row strides and pointers off 16 bytes
def test_append_rotates_and_quantises(h, hkv, hd, batch, odd):
    from glacier_b200 import ops
    rng = np.random.default_rng(h * 1000 + batch)
    width, layers, P = (h + 2 * hkv) * hd, 3, 600
    x = rng.standard_normal((batch, width + 3), dtype=np.float32) * 2
    bias = rng.standard_normal(width, dtype=np.float32)
    ang = rng.random((P, hd // 2)) * 6.3
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    pos = rng.integers(0, P, batch).astype(np.int32)
    slots = rng.permutation(16 * 40)[:batch].astype(np.int64)
    if batch > 2:
        slots[1] = -1
    pages = dev(rng.integers(0, 256, (40, ops.kv_q4_page_bytes(layers, hkv, hd)), dtype=np.uint8))
    t = dev(x)[:, 1:1 + width] if odd else dev(x[:, 1:1 + width])
    q = host(ops.qkv_rope_append_q4(t, dev(bias), dev(cos), dev(sin), dev(pos), dev(slots), h, hkv, hd, pages, layers,
                                    2))
    k, v = (host(a) for a in ops.kv_q4_read(pages, dev(slots), layers, 2, hkv, hd))
    y = (x[:, 1:1 + width] + bias).reshape(batch, h + 2 * hkv, hd)
    c, s = cos[pos][:, None], sin[pos][:, None]
    a, b = y[:, :h + hkv, :hd // 2], y[:, :h + hkv, hd // 2:]
    r32 = np.concatenate((a * c - b * s, a * s + b * c), -1)  # float32, each operation rounded
    r64 = np.concatenate((a.astype(np.float64) * c - b.astype(np.float64) * s,
                          a.astype(np.float64) * s + b.astype(np.float64) * c), -1)
    size = np.concatenate((np.abs(a) + np.abs(b),) * 2, -1)
    for i in range(batch):
        if slots[i] < 0:
            assert not q[i].any() and not k[i].any() and not v[i].any()
            continue
        assert (np.abs(q[i].reshape(h, hd) - r64[i, :h]) <= 3 * 2.0 ** -24 * size[i, :h]).all()
        np.testing.assert_array_equal(k[i], np.concatenate([held(r32[i, h + j]) for j in range(hkv)]))
        np.testing.assert_array_equal(v[i], np.concatenate([held(y[i, h + hkv + j]) for j in range(hkv)]))
    assert status_word() == 0


@gpu
def test_append_and_read_report_slots_and_positions_out_of_range():
    from glacier_b200 import ops
    h, hkv, hd = 4, 2, 64
    pages = dev(np.full((2, ops.kv_q4_page_bytes(1, hkv, hd)), 0x5A, np.uint8))
    x = torch.ones((4, (h + 2 * hkv) * hd), device="cuda")
    cos, sin = torch.ones((8, hd // 2), device="cuda"), torch.zeros((8, hd // 2), device="cuda")
    for slots, pos in (([32, -1, -1, -1], [0] * 4), ([-2, -1, -1, -1], [0] * 4), ([0, -1, -1, -1], [8, 0, 0, 0]),
                       ([0, -1, -1, -1], [-1, 0, 0, 0]), ([2 ** 40, -1, -1, -1], [0] * 4)):
        q = ops.qkv_rope_append_q4(x, None, cos, sin, dev(np.array(pos, np.int32)), dev(np.array(slots, np.int64)), h,
                                   hkv, hd, pages, 1, 0)
        assert not host(q).any()
        assert status_word() == 2
    assert (host(pages) == 0x5A).all()
    k, v = ops.kv_q4_read(pages, dev(np.array([32, -1], np.int64)), 1, 0, hkv, hd)
    assert not host(k).any() and not host(v).any() and status_word() == 2


# ---- page bookkeeping ----

def resize_ref(lens, targets, table, free, count, stride, rows):
    lens, table, free = list(lens), table.copy(), free.copy()
    lanes, max_pages = table.shape
    pg = lambda n: -(-n // 16)  # noqa: E731
    status = [0] * lanes
    valid = []
    for b in range(lanes):
        ok = 0 <= lens[b] <= 16 * max_pages and 0 <= targets[b] <= 16 * max_pages
        valid.append(ok and not (stride and targets[b] - lens[b] > stride))
    back = [table[b, j] for b in range(lanes) if valid[b] for j in range(pg(targets[b]), pg(lens[b]))]
    stack = list(free[:count]) + back[::-1]
    top = len(stack)
    free[:top] = stack
    out, wanted_pages, wanted_rows, used, off = [], 0, 0, 0, [0]
    new = list(lens)
    for b in range(lanes):
        got = []
        if not valid[b]:
            status[b] = EINVAL
        else:
            need, grow = max(0, pg(targets[b]) - pg(lens[b])), max(0, targets[b] - lens[b])
            wanted_pages += need
            wanted_rows += grow
            if (need and wanted_pages > top) or (grow and not stride and wanted_rows > rows):
                status[b] = ENOMEM
            else:
                for i in range(need):
                    table[b, pg(lens[b]) + i] = stack[top - 1 - used - i]
                used += need
                got = list(range(lens[b], targets[b]))
                new[b] = targets[b]
        cells = [(p, b, int(table[b, p // 16]) * 16 + p % 16) for p in got]
        out += cells + [(-1, -1, -1)] * (stride - len(cells) if stride else 0)
        off.append(len(out))
    out += [(-1, -1, -1)] * (rows - len(out))
    return new, table, free, top - used, status, np.array(out), off


RESIZES = {
    "one lane from nothing": dict(lens=[0], targets=[1]),
    "page borders": dict(lens=[0, 15, 16, 17, 31, 32], targets=[16, 16, 17, 32, 33, 49]),
    "unchanged and empty": dict(lens=[0, 5, 16, 0], targets=[0, 5, 16, 0]),
    "shrink and release": dict(lens=[40, 16, 33, 100, 1], targets=[33, 0, 32, 0, 0]),
    "pages of one lane go to another": dict(lens=[100, 0, 64, 0], targets=[0, 90, 1, 60], spare=0),
    "pages run out": dict(lens=[10, 0, 16, 5, 0], targets=[11, 40, 17, 6, 1], spare=2),
    "rows run out": dict(lens=[0, 0, 0, 3], targets=[20, 30, 5, 3], rows=27),
    "bad lengths": dict(lens=[5, -1, 4, 300, 7], targets=[6, 3, -2, 10, 10 ** 9], max_pages=8),
    "one row each": dict(lens=[0, 15, 16, 7, 47], targets=[1, 16, 17, 7, 40], stride=1),
    "three rows each, one too many": dict(lens=[0, 15, 16, 7], targets=[3, 16, 20, 9], stride=3),
    "a full house": dict(lens=[i * 7 % 50 for i in range(1024)], targets=[i * 13 % 60 for i in range(1024)]),
    "many rows": dict(lens=[0] * 37, targets=[(i * 397) % 1500 for i in range(37)]),
    "many padded rows": dict(lens=[3] * 9, targets=[(i * 97) % 1000 for i in range(9)], stride=1000),
}


@gpu
@pytest.mark.parametrize("name", list(RESIZES))
def test_resize(name):
    from glacier_b200 import ops
    c = RESIZES[name]
    rng = np.random.default_rng(len(name))
    lens, targets, stride = c["lens"], c["targets"], c.get("stride", 0)
    lanes = len(lens)
    sane = [n for n in lens + targets if 0 <= n < 10 ** 6]
    max_pages = c.get("max_pages", max(1, -(-max(sane) // 16)) + 1)
    held_pages = [-(-min(max(n, 0), 16 * max_pages) // 16) for n in lens]
    spare = c.get("spare", sum(-(-max(0, t) // 16) for t in targets if t < 10 ** 6) + 3)
    perm = rng.permutation(sum(held_pages) + spare).astype(np.int32)
    table = np.full((lanes, max_pages), -9, np.int32)
    at = 0
    for b, n in enumerate(held_pages):
        table[b, :n] = perm[at:at + n]
        at += n
    free = np.full(len(perm) + 2, -7, np.int32)
    free[:spare] = perm[at:]
    rows = lanes * stride if stride else c.get("rows", max(1, sum(max(0, t - n) for n, t in zip(lens, targets)
                                                                  if t < 10 ** 6)) + 5)
    t = dict(lens=dev(np.array(lens, np.int32)), table=dev(table), free=dev(free), count=dev(np.array([spare], np.int32)))
    i32 = dict(dtype=torch.int32, device="cuda")
    status, offsets = torch.full((lanes,), 99, **i32), torch.full((lanes + 1,), 99, **i32)
    pos, who = torch.full((rows,), 99, **i32), torch.full((rows,), 99, **i32)
    slots = torch.full((rows,), 99, dtype=torch.int64, device="cuda")
    ops.kv_resize(t["lens"], dev(np.array(targets, np.int32)), t["table"], t["free"], t["count"], status,
                  positions=pos, row_lanes=who, slots=slots, row_offsets=offsets, row_stride=stride)
    new, table2, free2, count2, st, cells, off = resize_ref(lens, targets, table, free, spare, stride, rows)
    assert host(status).tolist() == st
    assert host(t["lens"]).tolist() == new
    np.testing.assert_array_equal(host(t["table"]), table2)
    assert host(t["count"])[0] == count2
    np.testing.assert_array_equal(host(t["free"])[:count2], free2[:count2])
    np.testing.assert_array_equal(np.stack([host(pos), host(who), host(slots)], 1), cells)
    assert host(offsets).tolist() == off
    # back to where it was: the pages return so that the same growth takes the same ones again
    if all(s == 0 for s in st) and all(a <= b for a, b in zip(lens, targets)):
        ops.kv_resize(t["lens"], dev(np.array(lens, np.int32)), t["table"], t["free"], t["count"], status)
        assert host(t["lens"]).tolist() == lens and host(t["count"])[0] == spare
        np.testing.assert_array_equal(host(t["free"])[:spare], free[:spare])


@gpu
@pytest.mark.parametrize("seed", range(20))
def test_resize_of_random_batches(seed):
    """Any mixture of growth and release, with rows and without: pages and rows from a few to many per thread."""
    from glacier_b200 import ops
    rng = np.random.default_rng(500 + seed)
    lanes = 1024 if seed == 3 else int(np.exp(rng.uniform(0, np.log(700))))
    max_pages = int(np.exp(rng.uniform(0, np.log(max(2, min(2000, 60000 // lanes))))))
    kind = seed % 4
    some = lambda: rng.integers(0, 16 * max_pages + 1, lanes)  # noqa: E731
    lens = [some, lambda: 0 * some(), some, some][kind]()
    one_more = lambda: np.minimum(lens + rng.integers(0, 2, lanes), 16 * max_pages)  # noqa: E731
    targets = [some, some, lambda: 0 * some(), one_more][kind]()
    pg = -(-lens // 16)
    spare = int(rng.integers(0, max(2, int((-(-targets // 16)).sum()))) if seed % 5 == 0 else (-(-targets // 16)).sum())
    perm = rng.permutation(int(pg.sum()) + spare).astype(np.int32)
    table = np.full((lanes, max_pages), -9, np.int32)
    table[np.arange(max_pages) < pg[:, None]] = perm[:pg.sum()]
    free = np.full(len(perm) + 1, -7, np.int32)
    free[:spare] = perm[pg.sum():]
    rows = int(np.maximum(targets - lens, 0).sum()) + 3
    i32 = dict(dtype=torch.int32, device="cuda")
    new, table2, free2, count2, st, cells, off = resize_ref(lens.tolist(), targets.tolist(), table, free, spare, 0, rows)
    for with_rows in (False, True):
        if not with_rows and any(st):
            continue  # rows that run out are refused too: the same answer only when nothing does
        t = [dev(x) for x in (lens.astype(np.int32), table, free, np.array([spare], np.int32))]
        status = torch.full((lanes,), 99, **i32)
        pos, who = torch.full((rows,), 99, **i32), torch.full((rows,), 99, **i32)
        slots = torch.full((rows,), 99, dtype=torch.int64, device="cuda")
        more = dict(positions=pos, row_lanes=who, slots=slots) if with_rows else {}
        ops.kv_resize(t[0], dev(targets.astype(np.int32)), t[1], t[2], t[3], status, **more)
        assert host(status).tolist() == st and host(t[0]).tolist() == new and int(t[3]) == count2
        np.testing.assert_array_equal(host(t[1]), table2)
        np.testing.assert_array_equal(host(t[2])[:count2], free2[:count2])
        if with_rows:
            np.testing.assert_array_equal(np.stack([host(pos), host(who), host(slots)], 1), cells)


# ---- attention ----

CTX = {
    "one position": [1],
    "page borders": [15, 16, 17, 31, 32, 33, 47, 48, 49],
    "an empty lane among others": [5, 0, 64, 0, 200, 0],
    "all empty": [0, 0],
    "one long": [2111],
    "ragged": [1, 700, 33, 1290, 64, 2, 255, 16],
    "many short lanes": [(i * 37) % 90 for i in range(300)],
    "37 lanes alike": [333] * 37,
    "127 lanes nearly alike": [64 + i % 9 for i in range(127)],
    "128 lanes alike": [100] * 128,
    "129 lanes alike": [100] * 129,
    "lanes alike, some empty": [0 if i % 5 == 4 else 200 for i in range(90)],
}
HEADS = [(14, 2, 64), (28, 4, 128), (8, 8, 64), (3, 3, 128), (16, 2, 128), (5, 1, 64), (8, 2, 64), (6, 1, 128)]


def attention_case(rng, h, hkv, hd, ctxs, layers=2, layer=1):
    lanes = len(ctxs)
    max_pages = max(1, max(-(-c // 16) for c in ctxs)) + 1
    total = sum(-(-c // 16) for c in ctxs) + 2
    perm = rng.permutation(total)
    table = np.full((lanes, max_pages), 2 ** 30, np.int32)  # entries past a lane's pages name nothing
    at = 0
    for b, c in enumerate(ctxs):
        n = -(-c // 16)
        table[b, :n] = perm[at:at + n]
        at += n
    data = random_pool(rng, total, layers, hkv, hd)
    pool = Pool(data, layers, hkv, hd)
    # what lies behind a lane's last position is left over from others: NaN and infinite scales
    for b, c in enumerate(ctxs):
        for p in range(c, -(-c // 16) * 16):
            for j in range(hkv):
                blk = pool.block(table[b, p // 16], layer, j)
                for kind in (0, 1):
                    for g in range(hd // 32):
                        at = (16 + kind) * hd + 2 * (p % 16 // 2 * 2 * (hd // 32) + 2 * g + p % 2)
                        blk[at:at + 2] = np.frombuffer(np.float16([np.nan, np.inf][(p + g) % 2]).tobytes(), np.uint8)
    q = rng.standard_normal((lanes, h * hd), dtype=np.float32) * 1.5
    return q, pool, table


def check_attention(out, q, pool, table, ctxs, h, hkv, hd, layer=1, lanes=None):
    G = h // hkv
    for b in (range(len(ctxs)) if lanes is None else lanes):
        if ctxs[b] == 0:
            assert not out[b].any()
            continue
        for j in range(hkv):
            k, v = (pool.rows(table[b], ctxs[b], layer, j, kind) for kind in (0, 1))
            qs = q[b].reshape(h, hd)[j * G:(j + 1) * G]
            err = np.abs(out[b].reshape(h, hd)[j * G:(j + 1) * G] - attend64(qs, k, v)).max()
            assert err <= tolerance(qs, k, v), (b, j, err, tolerance(qs, k, v))


@gpu
@pytest.mark.parametrize("name", list(CTX))
@pytest.mark.parametrize("h,hkv,hd", HEADS[:4])
def test_attention_contexts(name, h, hkv, hd):
    from glacier_b200 import ops
    ctxs = CTX[name]
    rng = np.random.default_rng(len(name) + h)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd))
    lanes = None if len(ctxs) < 20 else list(range(0, len(ctxs), 29)) + [len(ctxs) - 1]
    if sum(ctxs) > 1000 and lanes is None:  # the layout is read cell by cell in Python: a few lanes suffice
        lanes = [b for b in range(len(ctxs)) if ctxs[b] < 800 or len(ctxs) == 1]
    check_attention(out, q, pool, table, ctxs, h, hkv, hd, lanes=lanes)
    assert status_word() == 0


@gpu
@pytest.mark.parametrize("h,hkv,hd", HEADS)
def test_attention_heads(h, hkv, hd):
    from glacier_b200 import ops
    ctxs = [77, 3, 160]
    rng = np.random.default_rng(h * hd)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs, layers=1, layer=0)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(1, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 1, 0, h, hkv, hd))
    check_attention(out, q, pool, table, ctxs, h, hkv, hd, layer=0)


@gpu
@pytest.mark.parametrize("scale_q", [1e-6, 30.0, 3e4])
def test_attention_of_tiny_and_huge_queries(scale_q):
    """A flat softmax, and ones that put all their weight on one position; one head of zeros."""
    from glacier_b200 import ops
    h, hkv, hd, ctxs = 7, 1, 128, [130]
    rng = np.random.default_rng(3)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    q = (q * np.float32(scale_q)).astype(np.float32)
    q[0, 2 * hd:3 * hd] = 0
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd))
    k, v = (pool.rows(table[0], ctxs[0], 1, 0, kind) for kind in (0, 1))
    for g in range(h):
        qs = q.reshape(h, hd)[g:g + 1]
        err = np.abs(out.reshape(h, hd)[g] - attend64(qs, k, v)[0]).max()
        assert err <= tolerance(qs, k, v), g


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_small_and_large_held_values(hd):
    """Scales over the format's whole range, mixed within a lane and from lane to lane."""
    from glacier_b200 import ops
    h, hkv, ctxs = 4, 2, [50, 50, 50]
    rng = np.random.default_rng(hd)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    for b, (lo, hi) in enumerate(((-21, -15), (8, 12.8), (-21, 12.8))):
        for page in table[b, :4]:
            for j in range(hkv):
                blk = pool.block(page, 1, j)
                for kind in (0, 1):
                    at = slice((16 + kind) * hd, (17 + kind) * hd)
                    s = np.ldexp(1.0, 0) * 2.0 ** rng.uniform(lo, hi, hd // 2)
                    step = np.maximum(2.0 ** (np.floor(np.log2(s)) - 6), 2.0 ** -21)
                    s = np.minimum(np.floor(s / step) * step, MAX_SCALE)
                    blk[at] = np.frombuffer(s.astype(np.float16).tobytes(), np.uint8)
                    assert (s.astype(np.float16).astype(np.float64) == s).all()
    q[1:] *= 1e-4
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd))
    check_attention(out, q, pool, table, ctxs, h, hkv, hd)


@gpu
def test_attention_poison_stays_in_its_lane_and_head():
    """A NaN scale makes the heads that attend it NaN, and nothing else."""
    from glacier_b200 import ops
    h, hkv, hd, ctxs = 8, 2, 64, [40, 40]
    rng = np.random.default_rng(8)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    bad = np.frombuffer(np.float16(np.nan).tobytes(), np.uint8)
    blk = pool.block(table[0, 1], 1, 0)  # lane 0, kv head 0, K of position 16 + 2, group 1
    blk[16 * hd + 2 * (1 * 4 + 2):][:2] = bad
    blk = pool.block(table[1, 0], 1, 1)  # lane 1, kv head 1, V of position 5, group 0
    blk[17 * hd + 2 * (2 * 4 + 1):][:2] = bad
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd))
    nan = np.isnan(out.reshape(2, hkv, h // hkv, hd))
    assert nan[0, 0].all() and not nan[0, 1].any() and not nan[1, 0].any()
    assert nan[1, 1][:, :32].all() and not nan[1, 1][:, 32:].any()


@gpu
def test_attention_clamps_the_context_and_leaves_out_bad_pages():
    from glacier_b200 import ops
    h, hkv, hd = 4, 2, 128
    rng = np.random.default_rng(12)
    q, pool, table = attention_case(rng, h, hkv, hd, [48, 64, 30])
    table = np.ascontiguousarray(table[:, :4])
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    run = lambda t, c: host(ops.paged_attention_q4(dev(q), pages, dev(t), dev(np.array(c, np.int32)), 2, 1, h, hkv, hd))  # noqa: E731
    good = run(table, [48, 64, 30])
    np.testing.assert_array_equal(run(table, [48, 2 ** 31 - 1, 30])[1], good[1])  # past the table: clamped
    np.testing.assert_array_equal(run(table, [48, 64, -5])[2], 0)
    assert status_word() == 0
    # lane 0 loses its middle page, lane 2 every page
    broken = table.copy()
    broken[0, 1], broken[2] = -1, 2 ** 31 - 1
    out = run(broken, [48, 64, 30])
    assert status_word() == 2
    np.testing.assert_array_equal(out[1], good[1])
    assert not out[2].any()
    keep = np.r_[0:16, 32:48]
    for j in range(hkv):
        k, v = (pool.rows(table[0], 48, 1, j, kind)[keep] for kind in (0, 1))
        qs = q[0].reshape(h, hd)[j * 2:j * 2 + 2]
        err = np.abs(out[0].reshape(h, hd)[j * 2:j * 2 + 2] - attend64(qs, k, v)).max()
        assert err <= tolerance(qs, k, v)


@gpu
def test_attention_is_the_same_every_time_and_on_any_stream():
    """Bit-identical results from a reused workspace, another stream, and a captured graph that is
    replayed on new inputs."""
    from glacier_b200 import ops
    h, hkv, hd, ctxs = 28, 4, 128, [500, 0, 1200, 17, 90]
    rng = np.random.default_rng(21)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    pages, t, c = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd))), dev(table), dev(np.array(ctxs, np.int32))
    qd, ws = dev(q), ops.paged_attention_q4_workspace(h, hkv, hd)
    args = (pages, t, c, 2, 1, h, hkv, hd)
    ref = host(ops.paged_attention_q4(qd, *args, workspace=ws))
    ws.fill_(float("nan"))
    np.testing.assert_array_equal(host(ops.paged_attention_q4(qd, *args, workspace=ws)), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = ops.paged_attention_q4(qd, *args, stream=side)
    side.synchronize()
    np.testing.assert_array_equal(out.cpu().numpy(), ref)
    graph = torch.cuda.CUDAGraph()
    qg, cg, og = qd.clone(), c.clone(), torch.empty_like(qd)
    with torch.cuda.graph(graph):
        ops.paged_attention_q4(qg, pages, t, cg, 2, 1, h, hkv, hd, out=og, workspace=ws)
    graph.replay()
    np.testing.assert_array_equal(host(og), ref)
    other = rng.standard_normal(q.shape, dtype=np.float32)
    qg.copy_(dev(other))
    cg.copy_(dev(np.array([16, 300, 7, 0, 33], np.int32).clip(0, np.array(ctxs, np.int32))))
    graph.replay()
    got = host(og)
    np.testing.assert_array_equal(got, host(ops.paged_attention_q4(dev(other), pages, t, cg, 2, 1, h, hkv, hd)))


@gpu
def test_attention_offsets_past_32_bits():
    """A pool of more than 4 GiB whose used pages lie at its far end."""
    from glacier_b200 import ops
    h, hkv, hd, ctxs, layers = 4, 1, 128, [40], 64
    rng = np.random.default_rng(5)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs, layers=layers, layer=63)
    pb = ops.kv_q4_page_bytes(layers, hkv, hd)
    n = (1 << 32) // pb + 40
    pages = torch.zeros((n, pb), dtype=torch.uint8, device="cuda")
    used = pool.data.reshape(-1, pb)
    pages[n - len(used):] = dev(used)
    t = np.where(table < len(used), table + (n - len(used)), table).astype(np.int32)
    out = host(ops.paged_attention_q4(dev(q), pages, dev(t), dev(np.array(ctxs, np.int32)), layers, 63, h, hkv, hd))
    check_attention(out, q, pool, table, ctxs, h, hkv, hd, layer=63)
    slot = torch.tensor([n * 16 - 1], device="cuda")
    x = torch.randn((1, (h + 2 * hkv) * hd), device="cuda")
    one = torch.ones((1, hd // 2), device="cuda")
    ops.qkv_rope_append_q4(x, None, one, one * 0, torch.zeros(1, dtype=torch.int32, device="cuda"), slot, h, hkv, hd,
                           pages, layers, 63)
    _, v = ops.kv_q4_read(pages, slot, layers, 63, hkv, hd)
    np.testing.assert_array_equal(host(v)[0], held(x[0, -hd:].cpu().numpy()))


# ---- longer and wider, against a vectorised reading of the format ----

def all_values(pool, layer):
    """float64 (K, V) [pages, hkv, 16, hd] of one layer of a Pool."""
    hkv, hd = pool.hkv, pool.hd
    blk = np.ascontiguousarray(np.asarray(pool.data).reshape(-1, pool.layers, hkv, 18 * hd)[:, layer])
    n, ng = len(blk), hd // 32
    k = blk[..., :8 * hd].reshape(n, hkv, 16, 4, ng, 4)  # [pos][t][g][byte]: dims 32g + 8t + 2 byte + nibble
    k = np.stack((k & 15, k >> 4), -1).transpose(0, 1, 2, 4, 3, 5, 6).reshape(n, hkv, 16, hd)
    v = blk[..., 8 * hd:16 * hd].reshape(n, hkv, 8, hd // 4, 2, 2)  # [pair][w][pos][byte]
    v = np.stack((v & 15, v >> 4), -1).transpose(0, 1, 2, 4, 3, 5, 6).reshape(n, hkv, 16, hd)
    s = np.ascontiguousarray(blk[..., 16 * hd:]).view(np.float16).reshape(n, hkv, 2, 8, ng, 2).astype(np.float64)
    s = s.transpose(2, 0, 1, 3, 5, 4).reshape(2, n, hkv, 16, ng).repeat(32, -1)
    return (k.astype(np.float64) - 7) * s[0], (v.astype(np.float64) - 7) * s[1]


@pytest.mark.parametrize("hd", [64, 128])
def test_the_vectorised_reading_agrees_with_the_one_by_cell(hd):
    pool = Pool(random_pool(np.random.default_rng(hd), 3, 2, 2, hd), 2, 2, hd)
    both = all_values(pool, 1)
    for kind in (0, 1):
        np.testing.assert_array_equal(both[kind][[2, 0], 1].reshape(32, hd), pool.rows([2, 0], 32, 1, 1, kind))


def check_all(out, q, pool, table, ctxs, h, hkv, hd):
    """check_attention for every lane, in 64 bits on the GPU."""
    G = h // hkv
    with np.errstate(invalid="ignore"):  # left-over scales are NaN and infinite
        k, v = (torch.from_numpy(x).cuda() for x in all_values(pool, 1))
    out, q = (torch.from_numpy(x).cuda().double().view(len(ctxs), hkv, G, hd) for x in (out, q))
    for b, c in enumerate(ctxs):
        if c == 0:
            assert not out[b].any()
            continue
        pages = torch.from_numpy(table[b, :-(-c // 16)].astype(np.int64)).cuda()
        kb, vb = (x[pages].transpose(0, 1).reshape(hkv, -1, hd)[:, :c] for x in (k, v))
        ref = torch.softmax(q[b] @ kb.transpose(1, 2) / hd ** 0.5, -1) @ vb
        size = (q[b].abs() @ kb.abs().transpose(1, 2)).amax((1, 2)) / hd ** 0.5
        tol = 2.0 ** -24 * (2 * (hd + 16) * size + 64) * vb.abs().amax((1, 2))
        err = (out[b] - ref).abs().amax((1, 2))
        assert (err <= tol).all(), (b, c, err, tol)


@gpu
@pytest.mark.parametrize("ctxs", [[24001], [9000, 0, 7777], [3000, 1, 5000, 16, 2999]])
@pytest.mark.parametrize("h,hkv,hd", [(14, 2, 64), (28, 4, 128), (4, 4, 128), (5, 1, 64), (8, 1, 128)])
def test_attention_of_few_lanes_with_long_contexts(h, hkv, hd, ctxs):
    from glacier_b200 import ops
    rng = np.random.default_rng(sum(ctxs) + h)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd))
    check_all(out, q, pool, table, ctxs, h, hkv, hd)


@gpu
@pytest.mark.parametrize("seed", range(24))
def test_attention_of_random_batches(seed):
    """Lane counts to 1024 and contexts of every spread: shares, pieces and cuts fall everywhere."""
    from glacier_b200 import ops
    rng = np.random.default_rng(1000 + seed)
    h, hkv, hd = HEADS[seed % len(HEADS)]
    lanes = 1024 if seed == 5 else int(np.exp(rng.uniform(0, np.log(500))))
    most = max(1, min(6000, 200000 // (lanes * hkv)))
    hi = int(np.exp(rng.uniform(0, np.log(most + 1))))
    ctxs = rng.integers(0, hi + 1, lanes)
    if seed % 3 == 0:
        ctxs[rng.integers(lanes)] = most  # one lane much longer than the others
    if seed % 4 == 1:
        ctxs[:] = hi
    ctxs = ctxs.tolist()
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd))
    check_all(out, q, pool, table, ctxs, h, hkv, hd)


@gpu
@pytest.mark.parametrize("h,hkv,hd", [(28, 4, 128), (8, 8, 64)])
def test_one_workspace_serves_every_shape_and_graph(h, hkv, hd):
    """Launches of different shapes, eager and replayed in turn, over a workspace that began with random bits."""
    from glacier_b200 import ops
    rng = np.random.default_rng(77)
    ws = ops.paged_attention_q4_workspace(h, hkv, hd)
    ws.view(torch.int32).random_(generator=torch.Generator("cuda").manual_seed(1))
    runs = []
    for ctxs in ([900, 0, 77], [4000], [100] * 40, list(range(1, 150)), [2500, 17] * 6):
        q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
        args = (dev(q), dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd))), dev(table),
                dev(np.array(ctxs, np.int32)), 2, 1, h, hkv, hd)
        ref = ops.paged_attention_q4(*args)
        out = torch.empty_like(ref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention_q4(*args, out=out, workspace=ws)
        runs.append((args, ref, out, graph))
    for i in rng.integers(0, 2 * len(runs), 200):
        args, ref, out, graph = runs[i // 2]
        out.zero_()
        if i % 2:
            graph.replay()
        else:
            ops.paged_attention_q4(*args, out=out, workspace=ws)
        assert torch.equal(out, ref)


@gpu
def test_append_read_and_resize_run_on_the_stream_they_are_given():
    from glacier_b200 import ops
    h, hkv, hd = 8, 2, 64
    i32 = dict(dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    lens, count, status = torch.zeros(3, **i32), torch.full((1,), 8, **i32), torch.full((3,), 9, **i32)
    table, free = torch.full((3, 4), -1, **i32), torch.arange(8, **i32)
    pos, who = torch.empty(3, **i32), torch.empty(3, **i32)
    slots = torch.empty(3, dtype=torch.int64, device="cuda")
    pages = torch.zeros((8, ops.kv_q4_page_bytes(1, hkv, hd)), dtype=torch.uint8, device="cuda")
    cos, sin = torch.ones((4, hd // 2), device="cuda"), torch.zeros((4, hd // 2), device="cuda")
    late, x = torch.zeros(3, **i32), torch.randn((3, (h + 2 * hkv) * hd), device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(50):  # work in front of the targets: another stream would see zeros
            torch.randn((2048, 2048), device="cuda") @ torch.randn((2048, 2048), device="cuda")
        late.fill_(1)
    ops.kv_resize(lens, late, table, free, count, status, positions=pos, row_lanes=who, slots=slots, row_stride=1,
                  stream=side)
    q = ops.qkv_rope_append_q4(x, None, cos, sin, pos, slots, h, hkv, hd, pages, 1, 0, stream=side)
    k, v = ops.kv_q4_read(pages, slots, 1, 0, hkv, hd, stream=side)
    side.synchronize()
    assert lens.tolist() == [1, 1, 1] and slots.tolist() == [7 * 16, 6 * 16, 5 * 16]
    assert torch.equal(q, x[:, :h * hd])
    for b in range(3):
        rows = x[b].cpu().numpy().reshape(-1, hd)
        np.testing.assert_array_equal(host(k)[b], np.concatenate([held(r) for r in rows[h:h + hkv]]))
        np.testing.assert_array_equal(host(v)[b], np.concatenate([held(r) for r in rows[h + hkv:]]))


# ---- together, as a decode loop uses them ----

@gpu
@pytest.mark.parametrize("h,hkv,hd", [(14, 2, 64), (28, 4, 128)])
def test_a_decode_loop_over_a_shared_pool(h, hkv, hd):
    """Requests of different ages grow position by position, end, and give their pages to new ones; every
    step's attention equals the 64-bit one over the rows that the requests appended themselves."""
    from glacier_b200 import ops
    rng = np.random.default_rng(h)
    lanes, max_pages, P, width = 3, 4, 64, (h + 2 * hkv) * hd
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = torch.full((7, ops.kv_q4_page_bytes(1, hkv, hd)), 0xEE, dtype=torch.uint8, device="cuda")
    table, free = torch.full((lanes, max_pages), -1, **i32), torch.arange(7, **i32)
    lens, count, status = torch.zeros(lanes, **i32), torch.tensor([7], **i32), torch.zeros(lanes, **i32)
    pos, who = torch.empty(lanes, **i32), torch.empty(lanes, **i32)
    slots = torch.empty(lanes, dtype=torch.int64, device="cuda")
    ang = np.arange(P)[:, None] * 1e4 ** (-np.arange(hd // 2) / (hd // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    kept = [[] for _ in range(lanes)]
    ends = [19, 33, 40]
    for step in range(45):
        target = [0 if len(kept[b]) >= ends[b] else len(kept[b]) + 1 for b in range(lanes)]
        ops.kv_resize(lens, dev(np.array(target, np.int32)), table, free, count, status, positions=pos,
                      row_lanes=who, slots=slots, row_stride=1)
        assert host(status).tolist() == [0] * lanes
        x = rng.standard_normal((lanes, width), dtype=np.float32)
        q = ops.qkv_rope_append_q4(dev(x), None, dev(cos), dev(sin), pos, slots, h, hkv, hd, pages, 1, 0)
        out = host(ops.paged_attention_q4(q, pages, table, lens, 1, 0, h, hkv, hd))
        qh = host(q)
        for b in range(lanes):
            if target[b] == 0:
                kept[b] = []
                assert not out[b].any()
                continue
            p = len(kept[b])
            y = x[b].reshape(-1, hd)
            a, c = y[h:h + hkv, :hd // 2], y[h:h + hkv, hd // 2:]
            k = np.concatenate((a * cos[p] - c * sin[p], a * sin[p] + c * cos[p]), -1)
            kept[b].append(([held(r) for r in k], [held(r) for r in y[h + hkv:]]))
            for j in range(hkv):
                ks, vs = (np.stack([r[i][j] for r in kept[b]]) for i in (0, 1))
                qs = qh[b].reshape(h, hd)[j * h // hkv:(j + 1) * h // hkv]
                err = np.abs(out[b].reshape(h, hd)[j * h // hkv:(j + 1) * h // hkv] - attend64(qs, ks, vs)).max()
                assert err <= tolerance(qs, ks, vs), (step, b, j)
    assert status_word() == 0


@gpu
@pytest.mark.parametrize("rows", [0, 128, 4096])
def test_resize_near_the_largest_stack(rows):
    """The stack's size and the pages given back add up to more than 2^31: what does not fit is dropped, what is
    taken comes from the top, and nothing lands in front of the stack."""
    from glacier_b200 import ops
    i32 = dict(dtype=torch.int32, device="cuda")
    capacity = 2 ** 31 - 1
    count, n = capacity - 5, 1000
    whole = torch.empty(4096 + capacity, **i32)  # the stack lies behind 4096 entries of ours
    front, free = whole[:4096], whole[4096:]
    front.fill_(-7)
    free[:4096] = -8
    free[count - 8:] = torch.arange(2000, 2013, **i32)
    table = torch.full((2, n), -9, **i32)
    table[0] = torch.arange(n, **i32)
    lens, targets = torch.tensor([16 * n, 0], **i32), torch.tensor([0, 128], **i32)
    counts, status = torch.tensor([count], **i32), torch.full((2,), 99, **i32)
    more = {}
    if rows:
        more = dict(positions=torch.empty(rows, **i32), row_lanes=torch.empty(rows, **i32),
                    slots=torch.empty(rows, dtype=torch.int64, device="cuda"))
    ops.kv_resize(lens, targets, table, free, counts, status, **more)
    assert status.tolist() == [0, 0] and lens.tolist() == [0, 128]
    taken = [995, 996, 997, 998, 999, 2007, 2006, 2005]  # the five that fitted, then three of the old top
    assert int(counts) == capacity - 8 and table[1, :9].tolist() == taken + [-9]
    assert free[count - 8:count - 3].tolist() == [2000, 2001, 2002, 2003, 2004]
    assert free[count:].tolist() == [999, 998, 997, 996, 995]
    assert (front == -7).all() and (free[:4096] == -8).all()
    if rows:
        assert more["slots"][:128].tolist() == [16 * p + r for p in taken for r in range(16)]
    # one lane of the longest block table that there can be, by many threads per lane
    del table
    n, count = 2 ** 26, capacity - 10
    table = torch.arange(n, **i32).view(1, n)
    lens, targets = torch.tensor([16 * n], **i32), torch.tensor([0], **i32)
    counts.fill_(count)
    free[count:] = -1
    if rows:
        more["positions"].fill_(5)
    ops.kv_resize(lens, targets, table, free, counts, status[:1], **more)
    assert int(status[0]) == 0 and int(lens) == 0 and int(counts) == capacity
    assert free[count:].tolist() == [n - 1 - k for k in range(10)]
    assert (front == -7).all() and (free[:4096] == -8).all()
    assert not rows or (more["positions"] == -1).all()


@gpu
@pytest.mark.parametrize("h,hkv,hd", [(4, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("exponent", [30, 60, 99, 115])
def test_attention_of_large_scores(h, hkv, hd, exponent):
    """Scores that are float32 numbers put all weight on one position, however large."""
    from glacier_b200 import ops
    ctx = 150
    rng = np.random.default_rng(exponent)
    q, pool, table = attention_case(rng, h, hkv, hd, [ctx])
    q = q.reshape(h, hd)
    q[:, 4:] = 0  # four dims: scores stay below 2^127
    q = np.ldexp(q / np.abs(q).max(1, keepdims=True), exponent).astype(np.float32) * np.float32(1.9)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q.reshape(1, -1)), pages, dev(table), dev(np.array([ctx], np.int32)), 2, 1, h,
                                      hkv, hd)).reshape(h, hd)
    for g in range(h):
        k, v = (pool.rows(table[0], ctx, 1, g // (h // hkv), kind) for kind in (0, 1))
        s = k @ q[g].astype(np.float64)
        best, second = np.argsort(s)[[-1, -2]]
        assert s[best] - s[second] > 2.0 ** -12 * np.abs(s).max()  # far above the scores' rounding, 2^-17
        assert np.abs(out[g] - v[best]).max() <= 2.0 ** -20 * np.abs(v).max(), g


# ---- weights far below the largest ----

@gpu
@pytest.mark.parametrize("h,hkv,hd,lanes,ctx", [(1, 1, 128, 1, 32), (7, 1, 64, 1, 64), (8, 8, 64, 64, 4000),
                                                (28, 4, 128, 100, 4000)])
def test_attention_counts_weights_far_below_the_largest(h, hkv, hd, lanes, ctx):
    """Position 0 is 22.2 nats (2^-32) above all others, and its V is zero: the output is what the others add.

    A weight is held to half a step of the smallest fp16 number, 2^-25, at 2^13 for the largest: 2^-38 of it
    each.  The 16 positions whose products one instruction sums with the largest weight's may lose all that lies
    2^-24 below its product's place.  Exponents near 32 have errors of 2^-19, two of them 2^-18."""
    from glacier_b200 import ops
    pages = -(-ctx // 16)
    blk = np.zeros((pages, hkv, 18 * hd), np.uint8)
    blk[..., :8 * hd] = 0x66  # K -1, V 1, scales 1
    blk[..., 8 * hd:16 * hd] = 0x88
    blk[..., 16 * hd:] = np.frombuffer(np.float16(1).tobytes() * hd, np.uint8)
    for q in range(hd // 4):  # position 0: K 0, V 0
        at = ((q % 8 // 2) * (hd // 32) + q // 8) * 4 + q % 2 * 2
        blk[0, :, at:at + 2] = 0x77
        blk[0, :, 8 * hd + q * 4:8 * hd + q * 4 + 2] = 0x77
    pool = Pool(blk.reshape(pages, -1), 1, hkv, hd)
    k, v = (pool.rows(list(range(pages)), 17, 0, hkv - 1, kind) for kind in (0, 1))
    assert not k[0].any() and not v[0].any() and (k[1:] == -1).all() and (v[1:] == 1).all()
    q = np.zeros((lanes, h, hd), np.float32)
    q[..., 5] = 22.2 * math.sqrt(hd)
    table = np.tile(np.arange(pages, dtype=np.int32), (lanes, 1))  # every lane reads the same pages
    out = host(ops.paged_attention_q4(dev(q.reshape(lanes, -1)), dev(pool.data.reshape(pages, -1)), dev(table),
                                      dev(np.full(lanes, ctx, np.int32)), 1, 0, h, hkv, hd))
    tail = (ctx - 1) * math.exp(-float(q[0, 0, 5]) / math.sqrt(hd))
    ref = tail / (1 + tail)
    assert np.abs(out - ref).max() <= ctx * 2.0 ** -38 + 16 * 2.0 ** -32 + 2.0 ** -18 * ref


@gpu
@pytest.mark.parametrize("h,hkv,hd", [(4, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("exponent", [116, 120, 124])
def test_attention_of_queries_near_float32s_largest(h, hkv, hd, exponent):
    """Scores that are float32 numbers put all weight on one position, whatever the size of q (below 2^125)."""
    from glacier_b200 import ops
    ctx = 150
    rng = np.random.default_rng(exponent)
    q, pool, table = attention_case(rng, h, hkv, hd, [ctx])
    q = q.reshape(h, hd)
    q[:, 4:] = 0  # four dims: scores stay below 2^127
    q = np.ldexp(q / np.abs(q).max(1, keepdims=True), exponent).astype(np.float32) * np.float32(1.9)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q.reshape(1, -1)), pages, dev(table), dev(np.array([ctx], np.int32)), 2, 1, h,
                                      hkv, hd)).reshape(h, hd)
    for g in range(h):
        k, v = (pool.rows(table[0], ctx, 1, g // (h // hkv), kind) for kind in (0, 1))
        s = k @ q[g].astype(np.float64)
        best, second = np.argsort(s)[[-1, -2]]
        assert s[best] - s[second] > 2.0 ** -12 * np.abs(s).max()  # far above the scores' rounding, 2^-17
        assert np.abs(out[g] - v[best]).max() <= 2.0 ** -20 * np.abs(v).max(), g


# ---- both fp16 parts of q and of the weights are there ----
# The tolerance above is a worst case, and a kernel without the low part of either operand would stay inside
# it.  Roundings that are independent add in squares: the n + 16 half steps of a score become sqrt(n + 16) of
# them, 8 more cover the weights' and sums' own, and a weighted mean of values whose weights are each off by such
# a relative error is off by the same in norm.  Over the heads of one kv head:
#
#     |out - ref|^2 <= sum_heads (2^-24 * (sqrt(n + 16) * max_p sum |q k| / sqrt(n) + 8))^2 |ref|^2
#
# One fp16 part alone has 11 bits: relative errors near 2^-13 for a weight or a q, 2 to 5 times the bound at least
# (the host model below).

NORM_CTX = {"few": [700, 64, 1290], "many": [200 + i * 53 % 900 for i in range(40)]}
NORM_HEADS = [(14, 2, 64), (8, 8, 64), (8, 2, 64), (28, 4, 128), (3, 3, 128), (16, 2, 128)]


def norm_excess(out, q, k, v):
    """|out - ref| over its bound, all heads of one kv head together."""
    n = q.shape[1]
    ref = attend64(q, k, v)
    size = (np.abs(q.astype(np.float64)) @ np.abs(k).T).max(1) / math.sqrt(n)
    bound = 2.0 ** -24 * (math.sqrt(n + 16) * size + 8) * np.linalg.norm(ref, axis=1)
    return np.linalg.norm(out - ref) / np.linalg.norm(bound)


def norm_case(name, h, hkv, hd):
    rng = np.random.default_rng(100 * len(name) + h + hd)
    q, pool, table = attention_case(rng, h, hkv, hd, NORM_CTX[name])
    with np.errstate(invalid="ignore"):
        k, v = all_values(pool, 1)

    def rows(b, j):
        c, ids = NORM_CTX[name][b], table[b, :-(-NORM_CTX[name][b] // 16)]
        return (q[b].reshape(hkv, h // hkv, hd)[j], k[ids, j].reshape(-1, hd)[:c], v[ids, j].reshape(-1, hd)[:c])
    return q, pool, table, rows


@gpu
@pytest.mark.parametrize("name", list(NORM_CTX))
@pytest.mark.parametrize("h,hkv,hd", NORM_HEADS)
def test_attention_error_in_norm(name, h, hkv, hd):
    from glacier_b200 import ops
    q, pool, table, rows = norm_case(name, h, hkv, hd)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    out = host(ops.paged_attention_q4(dev(q), pages, dev(table), dev(np.array(NORM_CTX[name], np.int32)), 2, 1, h, hkv,
                                      hd)).reshape(-1, hkv, h // hkv, hd)
    for b in range(len(out)):
        for j in range(hkv):
            assert norm_excess(out[b, j], *rows(b, j)) <= 1, (b, j)


@pytest.mark.parametrize("name", list(NORM_CTX))
@pytest.mark.parametrize("h,hkv,hd", NORM_HEADS)
def test_one_fp16_part_alone_is_outside_the_norm_bound(name, h, hkv, hd):
    """A host model of the kernel's operands, each of q and the weights in one part instead of two."""
    _, _, _, rows = norm_case(name, h, hkv, hd)
    worst_q, worst_p, both = [], [], []
    for b in range(len(NORM_CTX[name])):
        for j in range(hkv):
            q, k, v = rows(b, j)

            def model(q, part):
                s = q @ k.T / math.sqrt(hd)
                e = np.exp(s - s.max(1, keepdims=True)) * 128
                return part(e) @ v / e.sum(1, keepdims=True)
            one = lambda x: x.astype(np.float16).astype(np.float64)  # noqa: E731
            two = lambda x: one(x) + one(x - one(x))  # noqa: E731
            q64 = q.astype(np.float64)
            up = 2.0 ** (14 - np.floor(np.log2(np.abs(q64).max(1, keepdims=True))))  # as the kernel scales q
            worst_q.append(norm_excess(model(one(q64 * up) / up, two), q, k, v))
            worst_p.append(norm_excess(model(two(q64 * up) / up, one), q, k, v))
            both.append(norm_excess(model(two(q64 * up) / up, two), q, k, v))
    assert max(both) < 0.1
    assert max(worst_q) > 2 and max(worst_p) > 2


def test_no_rows_are_no_error():
    """An empty tensor's pointer is null: nothing to append or to read is not a missing argument."""
    a = dict(qkv=None, ld=768, bias=None, cos=4096, sin=4096, positions=64, pos=None, slots=None, batch=0, h=8, hkv=2,
             hd=64, q=None, ldq=512, pool=4096, num_pages=8, num_layers=2, layer=1)
    r = dict(pool=4096, num_pages=8, num_layers=2, layer=1, hkv=2, hd=64, slots=None, rows=0, k=None, v=None)
    assert capi("glacier_cuda_qkv_rope_append_q4", *a.values(), None) == 0
    assert capi("glacier_cuda_kv_q4_read_f32", *r.values(), None) == 0
    for over in (dict(hd=96), dict(layer=2), dict(pool=None)):  # the rest is checked all the same
        assert capi("glacier_cuda_qkv_rope_append_q4", *{**a, **over}.values(), None) == EINVAL
        assert capi("glacier_cuda_kv_q4_read_f32", *{**r, **over}.values(), None) == EINVAL


@gpu
def test_wrappers_take_no_rows():
    from glacier_b200 import ops
    h, hkv, hd = 8, 2, 64
    pages = torch.zeros((2, ops.kv_q4_page_bytes(1, hkv, hd)), dtype=torch.uint8, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    k, v = ops.kv_q4_read(pages, none, 1, 0, hkv, hd)
    assert k.shape == v.shape == (0, hkv * hd)
    cos = torch.ones((4, hd // 2), device="cuda")
    q = ops.qkv_rope_append_q4(torch.empty((0, (h + 2 * hkv) * hd), device="cuda"), None, cos, cos, none.int(), none, h,
                               hkv, hd, pages, 1, 0)
    assert q.shape == (0, h * hd) and not host(pages).any()


@gpu
def test_operators_on_another_stream_keep_what_the_caller_drops():
    """Inputs that are dropped after the call, and whose memory goes to other tensors, while the stream is busy."""
    from glacier_b200 import ops
    h, hkv, hd, ctxs = 8, 2, 64, [100, 37]
    rng = np.random.default_rng(31)
    q, pool, table = attention_case(rng, h, hkv, hd, ctxs)
    pages = dev(pool.data.reshape(-1, ops.kv_q4_page_bytes(2, hkv, hd)))
    lengths, t = dev(np.array(ctxs, np.int32)), dev(table)
    ref = host(ops.paged_attention_q4(dev(q), pages, t, lengths, 2, 1, h, hkv, hd))
    x = rng.standard_normal((2, (h + 2 * hkv) * hd), dtype=np.float32)
    one, zero = torch.ones((1, hd // 2), device="cuda"), torch.zeros((1, hd // 2), device="cuda")
    side = torch.cuda.Stream()
    args = [dev(q), t.clone(), lengths.clone()]
    more = [dev(x), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 17], device="cuda")]
    held_pages = torch.zeros_like(pages)
    grow = [torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([20, 5], dtype=torch.int32, device="cuda")]
    i32 = dict(dtype=torch.int32, device="cuda")
    blocks, free, count, status = torch.full((2, 4), -1, **i32), torch.arange(6, **i32), torch.tensor([6], **i32), torch.ones(2, **i32)
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = torch.randn((4096, 4096), device="cuda")
        for _ in range(60):
            a @ a
    out = ops.paged_attention_q4(args[0], pages, args[1], args[2], 2, 1, h, hkv, hd, stream=side)
    rot = ops.qkv_rope_append_q4(more[0], None, one, zero, more[1], more[2], h, hkv, hd, held_pages, 2, 1, stream=side)
    k, v = ops.kv_q4_read(held_pages, more[2], 2, 1, hkv, hd, stream=side)
    ops.kv_resize(grow[0], grow[1], blocks, free, count, status, stream=side)
    shapes = [(y.shape, y.dtype) for y in args + more + grow[1:]]
    del args, more, grow[1:]
    junk = [torch.full(s, 9, dtype=d, device="cuda") for s, d in shapes for _ in range(3)]
    side.synchronize()
    assert len(junk) == 21
    np.testing.assert_array_equal(out.cpu().numpy(), ref)
    np.testing.assert_array_equal(rot.cpu().numpy(), x[:, :h * hd])
    for b in range(2):
        rows = x[b].reshape(-1, hd)
        np.testing.assert_array_equal(k[b].cpu().numpy(), np.concatenate([held(r) for r in rows[h:h + hkv]]))
        np.testing.assert_array_equal(v[b].cpu().numpy(), np.concatenate([held(r) for r in rows[h + hkv:]]))
    assert status.tolist() == [0, 0] and grow[0].tolist() == [20, 5]
