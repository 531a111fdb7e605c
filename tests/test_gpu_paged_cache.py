"""The paged 8-bit decode cache on the GPU: block tables, rotary positions, cache write and read,
attention, and a decode loop of them together, against plain 64-bit forms (``_paged_ref``).

Tolerances.  A result rounded to type t is off by at most u = finfo(t).eps / 2 relative.  Integers,
codes and scales are exact (the scales are powers of two).  Rotation in fp32: angle to 2^-24 turns
after the 64-bit reduction, cosine and sine to 2 ulp, two products and a sum: 8 * 2^-24 of the pair's
norm.  Attention: operands in two fp16 terms (2^-22 relative), the tensor core's truncated sums over
D / 16 + 1 steps and an approximate exp2 (2^-22) put a logit off by at most
    delta = 2^-20 * scale * sum_i |q_i k_i| + 2^-20,
which moves the log-sum-exp by delta and the output by 2 delta max |v|.  For bf16 queries the weights
are one fp16 term instead: each p_j is off by at most 2^-11 p_j (11 significant bits, to nearest;
they stand at 2^9 or more for the largest, so what is subnormal, below 2^-14, is off by 2^-25, that is
2^-34 of the largest), which moves the output by at most sum_j 2^-11 p_j |v_j| + n 2^-34 max |v|.
"""

import math
import random

import pytest
import torch

import _paged_ref as ref
from submission_folder_b200 import ops
from submission_folder_b200.cache import PagedKVCache
from submission_folder_b200.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def half_ulp(t):
    return torch.finfo(t).eps / 2


# ---------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------
def _tables_state(rng, R, block, width, longest, blocks):
    lens = [rng.randint(0, longest) for _ in range(R)]
    order = list(range(blocks))
    rng.shuffle(order)
    tables = []
    for n in lens:
        need = -(-n // block)
        tables.append([order.pop() for _ in range(need)] + [-7] * (width - need))
    return lens, tables, order


@pytest.mark.parametrize("R,block,longest,extra,pad", [
    (1, 16, 40, 3, 0), (1, 1, 5, 9, 2), (7, 16, 100, 6, 3), (33, 32, 300, 40, 1), (16, 128, 3000, 2, 0),
    (1000, 16, 64, 500, 5), (1025, 64, 400, 900, 0), (8192, 16, 3, 8000, 0), (300, 17, 200, 300, 7),
])
def test_block_tables_follow_the_stack(dev, R, block, longest, extra, pad):
    """Three steps in place: tokens, idle rows, ended rows, prompts, rows too long for their
    table, and a pool that runs out."""
    rng = random.Random(R * 131 + block)
    width = -(-2 * longest // block) + 1
    lens, tables, free = _tables_state(rng, R, block, width, longest, -(-longest // block) * R + extra)
    cap = sum(-(-n // block) for n in lens) + len(free)
    t = ref.RefTables(lens, tables, free, block)
    i32 = dict(dtype=torch.int32, device=dev)
    d = [torch.tensor(x, **i32) for x in (lens, tables, free + [-1] * (cap - len(free)), [len(free)])]
    shift = [rng.randint(0, 200000) for _ in range(R)]
    for step in range(3):
        new = [rng.choice([1, 1, 0, -1, rng.randint(1, longest + 1), 2 * longest if step else 1]) for _ in range(R)]
        total = sum(max(x, 0) for x in new) + pad
        want = t.step(new, total, shift)
        got = ops.block_tables(d[0], torch.tensor(new, **i32), d[1], d[2], d[3], block, total,
                               shift=torch.tensor(shift, **i32))
        for name in ("lens", "cu", "slots", "positions", "granted"):
            assert getattr(got, name).tolist() == want[name], (step, name)
        assert got.lens is d[0] and d[0].tolist() == t.lens
        assert d[1].tolist() == t.tables
        n = int(d[3])
        assert n == len(t.free) and d[2][:n].tolist() == t.free


def test_block_tables_many_tokens_and_short_total(dev):
    """The cluster path (many tokens), rows of every size beside empty ones, and a ``total`` below
    the sum of the requests: the first tokens get their slots."""
    R, block = 50, 16
    rng = random.Random(5)
    new = [rng.choice([0, 1, 3, 700, 5000]) for _ in range(R)]
    need = sum(-(-n // block) for n in new)
    i32 = dict(dtype=torch.int32, device=dev)
    for total in (sum(new), sum(new) + 100, sum(new) - 3001, 0):
        lens, tables = torch.zeros(R, **i32), torch.full((R, 400), -7, **i32)
        free, count = torch.arange(need, **i32), torch.tensor([need], **i32)
        t = ref.RefTables([0] * R, tables.tolist(), free.tolist(), block)
        want = t.step(new, total, [0] * R)
        out = torch.empty_like(lens), torch.empty_like(count)
        for _ in range(2):    # without in-place lengths the step can be repeated
            got = ops.block_tables(lens, torch.tensor(new, **i32), tables, free, count, block, total, lens_out=out[0],
                                   free_count_out=out[1])
            assert got.slots.tolist() == want["slots"] and got.positions.tolist() == want["positions"]
            assert got.lens.tolist() == want["lens"] and int(got.free_count) == 0 and int(count) == need
            assert tables.tolist() == t.tables and lens.tolist() == [0] * R


def test_block_tables_release_feeds_admission(dev):
    """Blocks of a request that ends are taken by one that begins in the same step."""
    i32 = dict(dtype=torch.int32, device=dev)
    lens, tables = torch.tensor([40, 0], **i32), torch.tensor([[4, 2, 7, -1], [-1, -1, -1, -1]], **i32)
    free, count = torch.full((8,), -1, **i32), torch.zeros(1, **i32)
    s = ops.block_tables(lens, torch.tensor([-1, 33], **i32), tables, free, count, 16, 33)
    assert lens.tolist() == [0, 33] and tables[1, :3].tolist() == [7, 2, 4] and int(count) == 0
    assert s.slots.tolist() == [7 * 16 + i for i in range(16)] + [2 * 16 + i for i in range(16)] + [4 * 16]
    assert s.granted.tolist() == [0, 33]


@pytest.mark.parametrize("R,total", [(3, 8000), (600, 4000), (20, 100)])
@pytest.mark.parametrize("ask", [2 ** 31 - 1, 2 ** 31 - 100, 1 << 28])
def test_block_tables_refused_request_of_nearly_2_31_tokens(dev, R, total, ask):
    """Its rows say -1 and their positions; the requests before it and after it (for which the step has no
    rows) get what they get without it.  Several CTAs for each request, one, and one for all."""
    i32 = dict(dtype=torch.int32, device=dev)
    block, width, rng = 16, 6, random.Random(R)
    lens, tables, free = _tables_state(rng, R, block, width, 40, 4 * R)
    new = [rng.choice([1, 0, 33, -1]) for _ in range(R)]
    big = R // 3
    lens[big], new[big] = 5, total + (width + 1) * block
    cap = sum(-(-n // block) for n in lens) + len(free)
    t = ref.RefTables(lens, tables, free, block)
    shift = [rng.randint(0, 200000) for _ in range(R)]
    d = [torch.tensor(x, **i32) for x in (lens, tables, free + [-1] * (cap - len(free)), [len(free)])]
    want = t.step(new, total, shift)
    new[big] = ask
    got = ops.block_tables(d[0], torch.tensor(new, **i32), d[1], d[2], d[3], block, total, shift=torch.tensor(shift, **i32))
    for name in ("lens", "slots", "positions", "granted"):
        assert getattr(got, name).tolist() == want[name], name
    cu = [0]
    for n in new:
        cu.append(min(cu[-1] + max(n, 0), 2 ** 31 - 1))
    assert got.cu.tolist() == cu and d[1].tolist() == t.tables
    assert int(d[3]) == len(t.free) and d[2][:len(t.free)].tolist() == t.free


def test_block_tables_refusals(dev):
    i32 = dict(dtype=torch.int32, device=dev)
    a = dict(lens=torch.zeros(3, **i32), new=torch.ones(3, **i32), tables=torch.zeros(3, 2, **i32),
             free_list=torch.arange(4, **i32), free_count=torch.tensor([4], **i32), block_size=16, total=3)
    for name, bad, err in [("lens", torch.zeros(3, device=dev), ValueError), ("new", torch.ones(4, **i32), ValueError),
                           ("tables", torch.zeros(2, 2, **i32), ValueError), ("free_count", torch.zeros(2, **i32), ValueError),
                           ("block_size", 0, RuntimeError), ("total", -1, ValueError), ("lens", torch.zeros(3, dtype=torch.int32), RuntimeError),
                           ("shift", torch.zeros(3, dtype=torch.int64, device=dev), ValueError)]:
        with pytest.raises(err):
            ops.block_tables(**{**a, name: bad})
    with pytest.raises(RuntimeError, match="geometry"):
        ops.block_tables(**{**a, "tables": torch.zeros(1, 2, **i32).expand(3, 2)})
    one = {x: a[x][:1] for x in ("lens", "new", "tables")}
    assert ops.block_tables(**{**a, **one, "total": 1}).granted.tolist() == [1]     # a single row has any stride
    big = torch.zeros(8193, **i32)
    with pytest.raises(RuntimeError, match="8192"):
        ops.block_tables(big, big, torch.zeros(8193, 1, **i32), a["free_list"], a["free_count"], 16, 0)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def _rot_check(got, x, pos, f, inter, factor, inverse):
    want = ref.rotary(x, pos, f, inter, factor, inverse)
    u = half_ulp(x.dtype)
    d = 2 * f.numel()
    # the pair's norm bounds the fp32 part of the error
    h = x[..., :d].double()
    a, b = (h[..., 0::2], h[..., 1::2]) if inter else (h[..., :d // 2], h[..., d // 2:])
    norm = (a.square() + b.square()).sqrt() * factor
    norm = torch.stack([norm, norm], -1).flatten(-2) if inter else torch.cat([norm, norm], -1)
    tol = u * want[..., :d].abs() + 8 * 2.0 ** -24 * norm * (1 + u) + torch.finfo(x.dtype).smallest_normal * u * 2
    assert torch.all((got[..., :d].double() - want[..., :d]).abs() <= tol)
    assert torch.equal(got[..., d:], x[..., d:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,Hk,D,d", [(1, 32, 8, 128, 128), (16, 32, 8, 128, 64), (5, 3, 1, 80, 80), (7, 2, 2, 64, 58),
                                        (200, 4, 2, 128, 32), (1500, 8, 2, 128, 128), (3, 1, 1, 2, 2), (2, 5, 0, 96, 24),
                                        (1027, 7, 1, 256, 250)])
def test_rotary(dev, dtype, inter, T, H, Hk, D, d):
    g = torch.Generator(device=dev).manual_seed(T + d)
    q = torch.randn(T, H, D, generator=g, device=dev).to(dtype)
    k = torch.randn(T, Hk, D, generator=g, device=dev).to(dtype) if Hk else None
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=dev)
    pos[0] = 0
    f, _ = rotary_frequencies(d, device=dev)
    for inverse, factor in ((False, 1.0), (True, 1.25)):
        qo, ko = ops.rotary(q, k, pos, f, interleaved=inter, factor=factor, inverse=inverse)
        _rot_check(qo, q, pos, f, inter, factor, inverse)
        if Hk:
            _rot_check(ko, k, pos, f, inter, factor, inverse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rotary_strides_and_in_place(dev, dtype, offset):
    """Queries and keys as slices of one projection (odd offsets take the element-wise path), and
    in place; the values beside them stay."""
    T, H, Hk, D = 11, 4, 2, 64
    g = torch.Generator(device=dev).manual_seed(3)
    buf = torch.randn(T, (H + 2 * Hk) * D + 24, generator=g, device=dev).to(dtype)
    keep = buf.clone()
    q = buf[:, offset:offset + H * D].unflatten(1, (H, D))
    k = buf[:, offset + H * D:offset + (H + Hk) * D].unflatten(1, (Hk, D))
    pos = torch.randint(0, 9000, (T,), generator=g, device=dev)
    f, _ = rotary_frequencies(48, device=dev)
    qo, ko = ops.rotary(q, k, pos, f)
    assert qo.is_contiguous() and torch.equal(buf, keep)
    _rot_check(qo, q, pos, f, False, 1.0, False)
    _rot_check(ko, k, pos, f, False, 1.0, False)
    ops.rotary(q, k, pos, f, out=(q, k))
    assert torch.equal(q, qo) and torch.equal(k, ko)
    buf[:, offset:offset + (H + Hk) * D] = keep[:, offset:offset + (H + Hk) * D]
    assert torch.equal(buf, keep)


def test_rotary_far_and_negative_positions(dev):
    """2^40 turns are reduced without loss; a negative position turns back."""
    f, _ = rotary_frequencies(128, 500000.0, device=dev)
    pos = torch.tensor([1 << 20, (1 << 31) + 7, -5, -(1 << 22), 131071], device=dev)
    q = torch.randn(5, 2, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    got, _ = ops.rotary(q, None, pos, f)
    # 64-bit angle: position * f is rounded to 2^-53 relative, 2^31 rad * 2^-52 = 5e-7 rad
    want = ref.rotary(q, pos, f, False, 1.0, False)
    assert float((got.double() - want).abs().max()) < (8 * 2.0 ** -24 + 2 * 2.0 ** 31 * 2.0 ** -52) * 8


@pytest.mark.parametrize("inter", [False, True])
def test_rotary_inverse_is_the_gradient(dev, inter):
    """d <g, R q> / dq = R^T g: against the formula through autograd in float64, and against
    differences of the kernel itself (the map is linear, so a difference is exact up to rounding)."""
    g = torch.Generator(device=dev).manual_seed(9)
    q = torch.randn(6, 2, 64, generator=g, device=dev)
    w = torch.randn(6, 2, 64, generator=g, device=dev)
    pos = torch.randint(0, 100000, (6,), generator=g, device=dev)
    f, _ = rotary_frequencies(40, device=dev)
    grad, _ = ops.rotary(w, None, pos, f, interleaved=inter, factor=1.5, inverse=True)
    qq = q.double().requires_grad_()
    d = 40
    angle = pos.double()[:, None] * f
    c, s = 1.5 * angle.cos()[:, None], 1.5 * angle.sin()[:, None]
    a, b = (qq[..., :d:2], qq[..., 1:d:2]) if inter else (qq[..., :d // 2], qq[..., d // 2:d])
    x, y = a * c - b * s, b * c + a * s
    wx, wy = (w[..., :d:2], w[..., 1:d:2]) if inter else (w[..., :d // 2], w[..., d // 2:d])
    ((x * wx.double()).sum() + (y * wy.double()).sum() + (qq[..., d:] * w[..., d:].double()).sum()).backward()
    assert float((grad.double() - qq.grad).abs().max()) <= 16 * 2.0 ** -24 * 1.5 * float(w.abs().max()) * 1.5
    for dim in (0, 3, 19, 20, 39, 40, 63):
        e = torch.zeros_like(q)
        e[..., dim] = 1.0
        hi, _ = ops.rotary(q + e, None, pos, f, interleaved=inter, factor=1.5)
        lo, _ = ops.rotary(q - e, None, pos, f, interleaved=inter, factor=1.5)
        diff = ((hi.double() - lo.double()) * w.double()).sum(-1) / 2
        assert float((diff - grad[..., dim].double()).abs().max()) < 64 * 2.0 ** -23 * 1.5 * 64


def test_rotary_refusals(dev):
    q, k = torch.zeros(4, 2, 64, device=dev), torch.zeros(4, 1, 64, device=dev)
    pos, f = torch.zeros(4, dtype=torch.int64, device=dev), rotary_frequencies(64, device=dev)[0]
    for args, err in [((q.cpu(), k, pos, f), RuntimeError), ((q, k.half(), pos, f), ValueError), ((q, k[:3], pos, f), ValueError),
                      ((q, k, pos.int(), f), ValueError), ((q, k, pos[:3], f), ValueError), ((q, k, pos, f.float()), ValueError),
                      ((q, k, pos, torch.zeros(40, dtype=torch.float64, device=dev)), RuntimeError),
                      ((q.double(), None, pos, f), TypeError), ((q[0], None, pos, f), ValueError),
                      ((q.transpose(1, 2), None, pos, f), ValueError), ((q.clone().requires_grad_(), k, pos, f), RuntimeError)]:
        with pytest.raises(err):
            ops.rotary(*args)
    with pytest.raises(ValueError):
        ops.rotary(q, k, pos, f, out=(torch.empty_like(q), None))
    assert ops.rotary(q[:0], k[:0], pos[:0], f)[0].shape == (0, 2, 64)


# ---------------------------------------------------------------------------
# cache write and read
# ---------------------------------------------------------------------------
def _pool(dev, blocks, heads, block, dim, fmt, layout="hnd"):
    """(k_cache, v_cache, k_scale, v_scale) full of bytes that read as NaN in e4m3, scales NaN."""
    def codes():
        if layout == "hnd":
            c = torch.full((blocks, heads, block, dim), 0x7f, dtype=torch.uint8, device=dev)
        elif layout == "nhd":
            c = torch.full((blocks, block, heads, dim), 0x7f, dtype=torch.uint8, device=dev).transpose(1, 2)
        else:     # a wider row than the head: strides that nothing else has
            c = torch.full((blocks, heads, block + 3, dim + 16), 0x7f, dtype=torch.uint8, device=dev)[:, :, :block, :dim]
        return c.view(fmt)
    s = [torch.full((blocks, heads), math.nan, device=dev) for _ in range(2)]
    return codes(), codes(), s[0], s[1]


def _codes64(c):
    return c.to(torch.float32).double().cpu()


def _check_pool(pool, refs, dim):
    """Every code and scale that the reference holds is in the pool, exactly."""
    for cache, scale, r in ((pool[0], pool[2], refs[0]), (pool[1], pool[3], refs[1])):
        got, sc = _codes64(cache), scale.double().cpu()
        for (b, h), want in r.scale.items():
            assert sc[b, h] == want or (math.isnan(want) and torch.isnan(sc[b, h])), (b, h)
            for p, c in r.codes[b, h].items():
                assert torch.equal(got[b, h, p], c), (b, h, p)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,block,heads,layout", [(128, 16, 2, "hnd"), (64, 32, 3, "nhd"), (128, 128, 1, "odd"), (64, 64, 2, "hnd")])
def test_cache_write_prompts_and_appends(dev, fmt, dtype, dim, block, heads, layout):
    """Three sequences in one call, then appends of 1, 3 and ``block`` tokens whose magnitudes
    grow and shrink, so that scales rise, stay, and begin anew."""
    g = torch.Generator().manual_seed(dim + block)
    blocks = 24
    pool = _pool(dev, blocks, heads, block, dim, fmt, layout)
    refs = [ref.RefCache(heads, block, fmt) for _ in range(2)]
    order = torch.randperm(blocks, generator=g).tolist()
    tables, lens = [order[:8], order[8:16], order[16:]], [0, 0, 0]
    for n, size in ((block + 5, 1.0), (1, 0.3), (1, 9.0), (3, 70.0), (block, 0.01), (2, 3e4 if dtype != torch.float16 else 2e2)):
        slots = []
        for r in range(3):
            m = n + r if n > 3 else n
            for i in range(lens[r], lens[r] + m):
                slots.append(tables[r][i // block] * block + i % block)
            lens[r] += m
        x = [(torch.randn(len(slots), heads, dim, generator=g) * size).to(dtype) for _ in range(2)]
        ops.cache_write(x[0].to(dev), x[1].to(dev), *pool, torch.tensor(slots, device=dev))
        for r, xx in zip(refs, x):
            r.write(xx.double(), slots)
        _check_pool(pool, refs, dim)
    every = [tables[r][i // block] * block + i % block for r in range(3) for i in range(lens[r])]
    for out in DTYPES:
        k, v = ops.cache_read(*pool, torch.tensor(every + [-1, blocks * block], device=dev), out)
        assert not k[-2:].any() and not v[-2:].any()
        for got, r in ((k, refs[0]), (v, refs[1])):
            assert torch.equal(got[:-2].cpu(), r.read(every, dim).to(out))


def test_cache_write_long_list(dev):
    """More than 1024 tokens: pieces of the list that cut through blocks, sequences that begin
    anywhere in a piece, padding between them."""
    g = torch.Generator().manual_seed(2)
    heads, dim, block = 2, 64, 16
    lens = [1, 300, 17, 5, 700, 16, 33, 200]
    blocks = sum(-(-n // block) for n in lens)
    order = torch.randperm(blocks, generator=g).tolist()
    slots = []
    for n in lens:
        t = [order.pop() for _ in range(-(-n // block))]
        slots += [t[i // block] * block + i % block for i in range(n)] + [-1] * (n % 3)
    pool, refs = _pool(dev, blocks, heads, block, dim, E4M3), [ref.RefCache(heads, block, E4M3) for _ in range(2)]
    x = [torch.randn(len(slots), heads, dim, generator=g).bfloat16() for _ in range(2)]
    ops.cache_write(x[0].to(dev), x[1].to(dev), *pool, torch.tensor(slots, device=dev))
    for r, xx in zip(refs, x):
        r.write(xx.double(), slots)
    _check_pool(pool, refs, dim)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_cache_write_special_values(dev, fmt):
    """Zeros, the smallest numbers, the borders of the scale, a NaN and infinities: a block and
    head that holds one reads as NaN, the others are untouched by it; a fresh start clears it."""
    block, dim = 16, 64
    big = ref.LARGEST[fmt]
    rows = torch.zeros(8, 2, dim)
    rows[1, 0, 3] = 1e-45
    rows[2, 0, 5] = big * 2.0 ** -7                       # the border itself keeps the smaller scale
    rows[3, 0, 5] = torch.nextafter(torch.tensor(big * 2.0 ** -7), torch.tensor(1e9))
    rows[4, 0, 0] = math.nan
    rows[5, 1, 7] = -math.inf
    rows[6, 0, :] = torch.linspace(-3.4e38, 3.4e38, dim)
    rows[7, 1, :] = 1e-39                                 # subnormal
    slots = [i * block for i in range(8)]
    pool, refs = _pool(dev, 8, 2, block, dim, fmt), [ref.RefCache(2, block, fmt) for _ in range(2)]
    ops.cache_write(rows.to(dev), -rows.to(dev), *pool, torch.tensor(slots, device=dev))
    refs[0].write(rows.double(), slots)
    refs[1].write(-rows.double(), slots)
    _check_pool(pool, refs, dim)
    k, _ = ops.cache_read(*pool, torch.tensor(slots, device=dev), torch.float32)
    assert torch.isnan(k[4, 0]).all() and not torch.isnan(k[4, 1]).any() and torch.isnan(k[5, 1]).all()
    more = torch.ones(1, 2, dim)
    ops.cache_write(more.to(dev), more.to(dev), *pool, torch.tensor([4 * block + 1], device=dev))
    assert torch.isnan(pool[2][4, 0]) and pool[2][4, 1] > 0      # an append does not hide it
    ops.cache_write(more.to(dev), more.to(dev), *pool, torch.tensor([4 * block], device=dev))
    assert not torch.isnan(pool[2][4]).any()


def test_cache_write_same_slot_twice_and_strided_rows(dev):
    """Of a slot named twice among neighbours the last token stays; rows are slices of a
    projection."""
    block, dim, heads = 32, 128, 2
    g = torch.Generator().manual_seed(8)
    slots = [64, 65, 65, 64, 66, 70, 70, 70, 71]
    buf = torch.randn(len(slots), 3 * heads * dim, generator=g).bfloat16().to(dev)
    k, v = (buf[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in (1, 2))
    pool, refs = _pool(dev, 4, heads, block, dim, E4M3), [ref.RefCache(heads, block, E4M3) for _ in range(2)]
    ops.cache_write(k, v, *pool, torch.tensor(slots, device=dev))
    refs[0].write(k.double().cpu(), slots)
    refs[1].write(v.double().cpu(), slots)
    _check_pool(pool, refs, dim)


@pytest.mark.parametrize("before,times", [(0, 40), (0, 300), (1200, 300)])
def test_cache_write_slots_named_again_and_again(dev, before, times):
    """A run far longer than its block (each slot's last token stays), in a short list and in a long
    one whose pieces it crosses; with the block's first place and without."""
    block, dim, heads = 16, 64, 2
    g = torch.Generator().manual_seed(times + before)
    ids = torch.randperm(100, generator=g).tolist()
    slots = [ids[2 + i // block] * block + i % block for i in range(before)]
    for low in (1, 0):
        slots += (ids[low] * block + torch.randint(low, block, (times,), generator=g)).tolist()
    pool, refs = _pool(dev, 100, heads, block, dim, E4M3), [ref.RefCache(heads, block, E4M3) for _ in range(2)]
    one = torch.ones(1, heads, dim)
    ops.cache_write(one.to(dev), one.to(dev), *pool, torch.tensor([ids[1] * block], device=dev))
    x = [torch.randn(len(slots), heads, dim, generator=g).bfloat16() for _ in range(2)]
    ops.cache_write(x[0].to(dev), x[1].to(dev), *pool, torch.tensor(slots, device=dev))
    for r, xx in zip(refs, x):
        r.write(one.double(), [ids[1] * block])
        r.write(xx.double(), slots)
    _check_pool(pool, refs, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("exponent", [-126, -60, -5, 0, 30, 126, 127])
@pytest.mark.parametrize("mantissa", [1.0, 1.0 + 2.0 ** -23, 1.3, 1.5, 2.0 - 2.0 ** -23])
def test_cache_append_to_scales_of_other_programs(dev, fmt, dtype, exponent, mantissa):
    """An append to a block whose scale is no power of two: the next one, or what the new rows need, takes its
    place, and the held codes are brought to it by the true ratio and rounded once."""
    block, dim, heads = 16, 64, 2
    g = torch.Generator().manual_seed(exponent + 200)
    old = float(torch.tensor(mantissa)) * 2.0 ** exponent         # as the fp32 scale holds it (1.3 is none)
    codes = [round_to.clamp(-ref.LARGEST[fmt], ref.LARGEST[fmt]) for round_to in
             (ref.round_code(torch.randn(heads, 3, dim, generator=g).double() * 100, fmt) for _ in range(2))]
    pool = _pool(dev, 2, heads, block, dim, fmt)
    for cache, scale, c in zip(pool[:2], pool[2:], codes):
        cache[1, :, :3] = c.float().to(dev).to(fmt)
        scale[1] = old
    loud = torch.tensor([0.5, 4.0])[:, None] * min(old, 2.0 ** 100 if dtype != torch.float16 else 64.0) * 100    # the second head's scale grows
    x = [(torch.randn(2, heads, dim, generator=g) * loud).to(dtype) for _ in range(2)]
    ops.cache_write(x[0].to(dev), x[1].to(dev), *pool, torch.tensor([block + 3, block + 4], device=dev))
    up = 2.0 ** exponent * (1 if mantissa == 1.0 else 2)
    for cache, scale, c, rows in zip(pool[:2], pool[2:], codes, x):
        got, sc = _codes64(cache)[1], scale[1].double().cpu()
        for h in range(heads):
            want = max(up, ref.block_scale(float(rows[:, h].abs().max()), fmt))
            if up > 2.0 ** 127 or not torch.isfinite(rows[:, h]).all():       # fp16 rows may hold an infinity
                assert torch.isnan(sc[h])
                continue
            assert sc[h] == want
            moved = c[h] * (old / want)                         # e4m3: a product in fp32; int8: exact until its one rounding
            held = c[h] if want == old else ref.round_code(moved if fmt == INT8 else moved.float().double(), fmt)
            assert torch.equal(got[h, :3], held) and torch.equal(got[h, 3:5], ref.round_code(rows[:, h].double() / want, fmt))


def test_cache_write_read_refusals(dev):
    pool = _pool(dev, 4, 2, 16, 64, E4M3)
    x, slots = torch.zeros(3, 2, 64, device=dev), torch.arange(3, device=dev)
    ok = (x, x, *pool, slots)
    for i, bad, err in [(0, x.double(), TypeError), (0, x[:2], ValueError), (0, x[:, :1], ValueError), (1, x.half(), ValueError),
                        (6, slots.int(), ValueError), (6, slots[:2], ValueError), (6, slots.cpu(), RuntimeError),
                        (2, pool[0].view(torch.uint8), TypeError), (2, pool[0][:3], ValueError), (4, pool[2][:3], ValueError),
                        (4, pool[2].double(), ValueError), (0, x.clone().requires_grad_(), RuntimeError)]:
        with pytest.raises(err):
            ops.cache_write(*ok[:i], bad, *ok[i + 1:])
    with pytest.raises(RuntimeError, match="aligned"):
        y = torch.zeros(3, 2, 65, device=dev)[..., 1:]
        ops.cache_write(y, y, *pool, slots)
    for shape in ((4, 2, 24, 64), (4, 2, 16, 96)):
        c = torch.zeros(shape, dtype=INT8, device=dev)
        with pytest.raises(RuntimeError):
            ops.cache_read(c, c, pool[2], pool[3], slots)
    with pytest.raises(TypeError):
        ops.cache_read(*pool, slots, torch.float64)
    assert ops.cache_read(*pool, slots[:0])[0].shape == (0, 2, 64)
    ops.cache_write(x[:0], x[:0], *pool, slots[:0])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention_case(dev, lens, heads, group, dim, block, fmt, dtype, queries, layout="hnd", spread=1.0, seed=0):
    """A pool written by the cache itself, its values read back as float64, queries, tables."""
    g = torch.Generator().manual_seed(seed + dim + block + sum(lens))
    need = [-(-n // block) for n in lens]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=g).tolist()
    pool = _pool(dev, blocks, heads, block, dim, fmt, layout)
    tables = torch.full((len(lens), max(need) + 2), blocks - 1, dtype=torch.int32)
    slots = []
    for r, n in enumerate(lens):
        ids = [order.pop() for _ in range(need[r])]
        tables[r, :need[r]] = torch.tensor(ids, dtype=torch.int32)
        slots += [ids[i // block] * block + i % block for i in range(n)]
    T = len(slots)
    slots = torch.tensor(slots, dtype=torch.int64, device=dev)
    size = torch.exp2(torch.randint(-2, 3, (T, 1, 1), generator=g).float() * spread)   # scales that differ by block
    k = (torch.randn(T, heads, dim, generator=g)).to(dtype).to(dev)
    v = (torch.randn(T, heads, dim, generator=g) * size).to(dtype).to(dev)
    ops.cache_write(k, v, *pool, slots)
    k, v = (x.double() for x in ops.cache_read(*pool, slots, torch.float32))
    q = (1.5 * torch.randn(sum(queries), heads * group, dim, generator=g)).to(dtype).to(dev)
    return pool, tables.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), q, k, v


def _attention_check(out, lse, q, k, v, lens, queries, scale, causal):
    u = half_ulp(q.dtype)
    a = b = 0
    for n, m in zip(lens, queries):
        qq, kk, vv = q[a:a + m].double(), k[b:b + n], v[b:b + n]
        want, wl = ref.attention(qq, kk, vv, scale, causal)
        if n:
            H, Hk = qq.shape[1], kk.shape[1]
            mass = torch.einsum("mhd,nhd->mhn", qq.abs(), kk.abs().repeat_interleave(H // Hk, 1)).amax(-1)
            delta = 2.0 ** -20 * abs(scale) * mass + 2.0 ** -20
            top = vv.abs().amax((0, 2)).repeat_interleave(H // Hk)
            tol = (2 * delta * top)[..., None]
            if q.dtype == torch.bfloat16:
                tol = tol + 2.0 ** -11 * ref.attention(qq, kk, vv.abs(), scale, causal)[0] + n * 2.0 ** -34 * top[:, None]
            tol = u * want.abs() + tol * (1 + u)
        else:
            delta, tol = torch.zeros_like(wl), torch.zeros_like(want)
        got, gl = out[a:a + m].double(), lse[a:a + m].double()
        assert torch.all((got - want).abs() <= tol), float(((got - want).abs() - tol).max())
        seen = torch.isfinite(wl)
        assert torch.equal(gl[~seen], wl[~seen])
        assert torch.all((gl - wl).abs()[seen] <= (delta + 2.0 ** -23 * wl.abs())[seen])
        a, b = a + m, b + n


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,group,dim,block,lens", [
    (8, 4, 128, 16, [1]), (8, 4, 128, 16, [512]), (2, 4, 128, 32, [31, 32, 33, 1, 0, 64, 65, 15, 16, 17]),
    (1, 8, 64, 16, [4097]), (3, 1, 128, 64, [700, 3, 0, 0, 129]), (4, 2, 64, 128, [127, 128, 129, 1000]),
    (2, 7, 128, 16, [2000, 5]), (1, 16, 128, 32, [900]), (1, 40, 64, 32, [300, 7]), (8, 4, 128, 64, [20000]),
])
def test_attention_single_tokens(dev, fmt, dtype, heads, group, dim, block, lens):
    pool, tables, n, q, k, v = _attention_case(dev, lens, heads, group, dim, block, fmt, dtype, [1] * len(lens))
    out, lse = ops.cache_attention(q, *pool, tables, n, want_lse=True)
    _attention_check(out, lse, q, k, v, lens, [1] * len(lens), dim ** -0.5, True)
    again = ops.cache_attention(q, *pool, tables, n)
    assert torch.equal(again, out)          # the same bits every time


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("fmt,dtype", [(E4M3, torch.bfloat16), (INT8, torch.float32)])
@pytest.mark.parametrize("heads,group,dim,block,lens,queries", [
    (2, 4, 128, 16, [40, 100, 3, 0, 1, 17], [4, 1, 5, 2, 0, 3]), (1, 1, 64, 32, [200, 33], [20, 33]),
    (8, 4, 128, 32, [1500], [4]), (2, 3, 128, 64, [64, 63, 300], [2, 7, 1]), (1, 5, 64, 16, [50], [50]),
])
def test_attention_several_tokens(dev, causal, fmt, dtype, heads, group, dim, block, lens, queries):
    """Several new tokens per sequence, more than the sequence has, none, and padding rows that
    are left alone."""
    pool, tables, n, q, k, v = _attention_case(dev, lens, heads, group, dim, block, fmt, dtype, queries)
    pad = 3
    q = torch.cat([q, torch.full_like(q[:1], math.nan).repeat(pad, 1, 1)])
    cu = torch.tensor([0] + queries, device=dev).cumsum(0).int()
    out = torch.full_like(q, 7.0)
    got, lse = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=max(queries), scale=0.1, causal=causal, want_lse=True,
                                   out=out)
    assert got is out and torch.all(out[-pad:] == 7.0)
    _attention_check(out, lse, q, k, v, lens, queries, 0.1, causal)


@pytest.mark.parametrize("layout", ["nhd", "odd"])
def test_attention_strides(dev, layout):
    """Caches of other layouts, queries and outputs as slices, a table that is a slice."""
    lens = [70, 5, 260]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 2, 4, 128, 16, E4M3, torch.bfloat16, [1] * 3, layout)
    wide = torch.zeros(3, 2 * tables.shape[1], dtype=torch.int32, device=dev)
    wide[:, :tables.shape[1]] = tables
    buf = torch.zeros(3, 3 * 8 * 128, dtype=torch.bfloat16, device=dev)
    qs = buf[:, 1024:2048].unflatten(1, (8, 128))
    qs.copy_(q)
    out = torch.zeros(8, 3, 128, dtype=torch.bfloat16, device=dev).transpose(0, 1)
    _, lse = ops.cache_attention(qs, *pool, wide[:, :tables.shape[1]], n, want_lse=True, out=out)
    _attention_check(out, lse, q, k, v, lens, [1] * 3, 128 ** -0.5, True)


def test_attention_value_scales_far_apart(dev):
    """Value scales over a range that fp16 weights alone could not carry."""
    lens = [300, 64]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 2, 4, 64, 16, E4M3, torch.float32, [1] * 2, spread=12.0)
    out, lse = ops.cache_attention(q, *pool, tables, n, want_lse=True)
    _attention_check(out, lse, q, k, v, lens, [1] * 2, 64 ** -0.5, True)


@pytest.mark.parametrize("times_k,times_v", [(1.0, 2.0 ** -115), (1.0, 2.0 ** 118), (1.3, 1.7), (0.7, 1.1 * 2.0 ** -100)])
def test_attention_scales_of_other_programs(dev, times_k, times_v):
    """Value scales at both ends of the normal range, and scales that are no powers of two: their
    logarithm is off by 2^-22 at most, their products with the codes by 2^-24, of the 2^-19 allowed."""
    lens = [300, 64]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 2, 4, 128, 32, INT8, torch.float32, [1] * 2)
    pool[2].mul_(times_k)
    pool[3].mul_(times_v)
    used = pool[3][torch.isfinite(pool[3])]
    assert used.min() >= 2.0 ** -126 and torch.isfinite(used * 127).all()
    out, lse = ops.cache_attention(q, *pool, tables, n, want_lse=True)
    _attention_check(out, lse, q, k * times_k, v * times_v, lens, [1] * 2, 128 ** -0.5, True)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [10, 23, 24, 25, 26, 27, 28, 40, 100])
def test_attention_logits_of_any_size(dev, power, dtype, sign):
    """Logits of 1.37 * 2^power and 0 (sign 1: two tokens of 3000 carry everything), or all alike and below
    zero (sign -1: all tokens carry the same), under value scales of 2^-12 to 2^12.  Equal logits are equal in any
    arithmetic, so the output is the plain mean of their values: off by the weights' rounding (2^-11 relative for
    bf16 queries, 2^-22 otherwise), what is subnormal in fp16 and the truncated sums, as in the header above."""
    heads, dim, block, n = 2, 64, 32, 3000
    g = torch.Generator().manual_seed(power)
    pool = _pool(dev, 95, heads, block, dim, E4M3)
    order = torch.randperm(94, generator=g)
    at = torch.arange(n)
    slots = (order[at // block] * block + at % block).to(dev)
    big = torch.tensor([700, 2222]) if sign > 0 else at
    k = torch.zeros(n, heads, dim)
    k[big, :, 5] = 2.0 ** power
    v = torch.randn(n, heads, dim, generator=g) * torch.exp2(torch.randint(-12, 13, (n // block + 1, 1, 1), generator=g).float())[at // block]
    ops.cache_write(k.to(dev), v.to(dev), *pool, slots)
    kk, vv = (x.double() for x in ops.cache_read(*pool, slots, torch.float32))
    assert torch.equal(kk.cpu(), k.double())
    q = torch.zeros(1, heads * 3, dim)
    q[:, :, 5] = 1.37
    q = q.to(dtype).to(dev)
    lens, table = torch.tensor([n], dtype=torch.int32, device=dev), order[None].int().to(dev)
    out, lse = ops.cache_attention(q, *pool, table, lens, scale=sign, want_lse=True)
    vv = vv[big.to(dev)].repeat_interleave(3, 1)
    want, mean = vv.mean(0), vv.abs().mean(0)
    tol = half_ulp(dtype) * want.abs() + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -18) * mean + n * 2.0 ** -34 * vv.abs().amax()
    assert torch.all((out[0].double() - want).abs() <= tol)
    logit = sign * float(q[0, 0, 5]) * 2.0 ** power
    assert torch.all((lse.double() - (logit + math.log(len(big)))).abs() <= 2.0 ** -21 * abs(logit) + 2.0 ** -20)


def _half_step(x, t):
    """Half the distance of the numbers of type t around x (float64), exactly."""
    _, e = torch.frexp(x)                                # |x| in [2^(e - 1), 2^e)
    return torch.finfo(t).eps / 2 * torch.exp2((e - 1).double())


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group,queries", [(128, 4, 1), (64, 4, 1), (128, 4, 3), (64, 2, 5)])
def test_attention_is_rounded_once(dev, dim, group, queries, dtype, fmt):
    """An output is its 64-bit value to half a step of its type, and little more: the weights carry 22 bits for
    every type of query.  With small logits delta of the header is 2^-20 (1 + scale * mass), which moves an output by
    2 delta sum_j p_j |v_j|; two fp16 terms put a weight off by 2^-22 of itself, or by 2^-25 where the second is subnormal,
    that is 2^-33 of the largest (at 2^8 or more), and a sum over at most 17 steps by 17 * 2^-24."""
    lens = [64, 200, 33, 512, 7, 100] * 8
    pool, tables, n, q, k, v = _attention_case(dev, lens, 4, group, dim, 16, fmt, dtype, [queries] * len(lens))
    q = (q.double() * 0.02).to(dtype)
    cu = torch.arange(0, queries * len(lens) + 1, queries, dtype=torch.int32, device=dev)
    out, lse = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=queries, want_lse=True)
    b, scale = 0, dim ** -0.5
    for r, m in enumerate(lens):
        qq, kk, vv = q[r * queries:(r + 1) * queries].double(), k[b:b + m], v[b:b + m]
        want, wl = ref.attention(qq, kk, vv, scale, True)
        mean, _ = ref.attention(qq, kk, vv.abs(), scale, True)
        mass = torch.einsum("mhd,nhd->mhn", qq.abs(), kk.abs().repeat_interleave(group, 1)).amax(-1)
        delta = 2.0 ** -20 * (1 + scale * mass)
        tol = (2 * delta + 2.0 ** -21 + 17 * 2.0 ** -24)[..., None] * mean + m * 2.0 ** -33 * vv.abs().amax()
        got, gl = out[r * queries:(r + 1) * queries].double(), lse[r * queries:(r + 1) * queries].double()
        off = (got - want).abs() - _half_step(want, dtype) - tol
        assert float(off.max()) <= 0, (r, m, float(off.max()))
        assert torch.all((gl - wl).abs() <= delta + 2.0 ** -23 * wl.abs())
        b += m


@pytest.mark.parametrize("fmt,dtype", [(E4M3, torch.bfloat16), (INT8, torch.float32)])
@pytest.mark.parametrize("heads,group,dim,block,lens,queries", [
    (8, 2, 64, 16, [150000, 900], [1, 1]), (8, 2, 64, 32, [300000], [1]), (4, 4, 128, 16, [70, 240000], [1, 3])])
def test_attention_long_pieces(dev, heads, group, dim, block, lens, queries, fmt, dtype):
    """Warps with more than 32 blocks of one unit, whose list of block ids is read on (16 steps of two blocks each, or
    32 steps of one).  On top of the header's bounds up to 80 steps' sums in fp32, each rounded by 2^-24."""
    warps = 148 * (12 if dim == 64 and dtype == torch.bfloat16 and max(queries) == 1 else 8)
    steps = sum(-(-n // 32) for n in lens) * heads // warps
    assert (32 * block) // 32 < steps <= 80
    pool, tables, n, q, k, v = _attention_case(dev, lens, heads, group, dim, block, fmt, dtype, queries)
    cu = torch.tensor([0] + queries, device=dev).cumsum(0).int()
    out, lse = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=max(queries), want_lse=True)
    a = b = 0
    for m, nq in zip(lens, queries):
        qq, kk, vv = q[a:a + nq].double(), k[b:b + m], v[b:b + m]
        want, wl = ref.attention(qq, kk, vv, dim ** -0.5, True)
        mean, _ = ref.attention(qq, kk, vv.abs(), dim ** -0.5, True)
        mass = torch.einsum("mhd,nhd->mhn", qq.abs(), kk.abs().repeat_interleave(group, 1)).amax(-1)
        delta = 2.0 ** -20 * (1 + dim ** -0.5 * mass) + 80 * 2.0 ** -24
        tol = (2 * delta)[..., None] * mean + m * 2.0 ** -33 * vv.abs().amax()
        assert torch.all((out[a:a + nq].double() - want).abs() <= _half_step(want, dtype) + tol)
        assert torch.all((lse[a:a + nq].double() - wl).abs() <= delta + 2.0 ** -23 * wl.abs())
        a, b = a + nq, b + m
    assert torch.equal(ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=max(queries)), out)


def test_attention_nan_and_bad_pages(dev):
    """A NaN block reaches the rows that see it and no others; a table entry outside the pool reads as
    NaN; queries with a NaN or an infinity stay in their row."""
    lens = [64, 64, 64]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 1, 2, 128, 16, INT8, torch.bfloat16, [4] * 3)
    cu = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=dev)
    clean, _ = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=4, want_lse=True)
    # sequence 0: the last block's values are NaN; with 4 new tokens every row sees the block
    bad = [t.clone() for t in pool]
    bad[3][tables[0, 3]] = math.nan
    out = ops.cache_attention(q, *bad, tables, n, cu=cu, max_q=4)
    assert torch.isnan(out[:4]).all() and torch.equal(out[4:], clean[4:])
    # 17 tokens: the second block holds only the last new token, which the first three rows do not see
    short = torch.tensor([17, 64, 64], dtype=torch.int32, device=dev)
    clean17 = ops.cache_attention(q, *pool, tables, short, cu=cu, max_q=4)
    bad = [t.clone() for t in pool]
    bad[2][tables[0, 1]] = math.nan
    out = ops.cache_attention(q, *bad, tables, short, cu=cu, max_q=4)
    assert torch.equal(out[:3], clean17[:3]) and torch.isnan(out[3]).all() and torch.equal(out[4:], clean17[4:])
    for page in (-1, 10 ** 6, -(2 ** 31)):
        t = tables.clone()
        t[1, 2] = page
        out = ops.cache_attention(q, *pool, t, n, cu=cu, max_q=4)
        assert torch.isnan(out[4:8]).all() and torch.equal(out[:4], clean[:4]) and torch.equal(out[8:], clean[8:])
    qq = q.clone()
    qq[5, 0, 3], qq[9, 1, 0] = math.nan, math.inf
    out = ops.cache_attention(qq, *pool, tables, n, cu=cu, max_q=4)
    assert torch.isnan(out[5, 0]).all() and torch.equal(out[5, 1], clean[5, 1]) and torch.isnan(out[9, 1]).all()
    keep = [i for i in range(12) if i not in (5, 9)]
    assert torch.equal(out[keep], clean[keep])


def test_attention_nan_values_that_nobody_sees(dev):
    """As the 17-token case above with NaN value scales: a block that holds only the last new token's values
    does not reach the rows that do not see it."""
    for fmt, dtype in ((INT8, torch.bfloat16), (E4M3, torch.float32)):
        lens = [17, 64, 64]
        pool, tables, n, q, k, v = _attention_case(dev, lens, 1, 2, 128, 16, fmt, dtype, [4] * 3)
        cu = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=dev)
        clean = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=4)
        pool[3][tables[0, 1]] = math.nan
        out, lse = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=4, want_lse=True)
        assert torch.equal(out[:3], clean[:3]) and torch.isnan(out[3]).all() and torch.equal(out[4:], clean[4:])
        assert torch.isfinite(lse).all()            # the keys are sound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_more_rows_than_max_q_is_nan(dev, dtype):
    """The rows of a sequence with more query tokens than the call allows for are marked, all of them; the
    other sequences are right and the padding is left alone."""
    lens, queries = [100, 40, 0, 70], [2, 5, 3, 1]      # the third sees nothing, however many rows it has
    pool, tables, n, q, k, v = _attention_case(dev, lens, 2, 4, 128, 16, E4M3, dtype, queries)
    q = torch.cat([q, q[:2]])
    cu = torch.tensor([0] + queries, device=dev).cumsum(0).int()
    out = torch.full_like(q, 7.0)
    got, lse = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=2, want_lse=True, out=out)
    assert torch.isnan(got[2:7]).all() and torch.isnan(lse[2:7]).all()
    assert not got[7:10].any() and torch.all(lse[7:10] == -math.inf)
    # the others by the header's bounds (a larger max_q cuts the line of work elsewhere, so that sums in fp32
    # come in another order: no other call gives the same bits)
    _attention_check(got[:2], lse[:2], q[:2], k[:100], v[:100], [100], [2], 128 ** -0.5, True)
    _attention_check(got[10:11], lse[10:11], q[10:11], k[140:], v[140:], [70], [1], 128 ** -0.5, True)
    assert torch.all(got[11:] == 7.0)


@pytest.mark.parametrize("pad", [1, 200])
def test_lse_of_padding_rows(dev, pad):
    """The log-sum-exp of rows of no sequence is -inf, whatever its memory held before."""
    queries = [2, 0, 1]
    pool, tables, n, q, k, v = _attention_case(dev, [40, 3, 5], 2, 4, 64, 16, INT8, torch.bfloat16, queries)
    q = torch.cat([q, q[:1].repeat(pad, 1, 1)])
    cu = torch.tensor([0] + queries, device=dev).cumsum(0).int()
    for _ in range(3):
        torch.full((q.shape[0], q.shape[1]), math.nan, device=dev)      # what the allocator gives next
        _, lse = ops.cache_attention(q, *pool, tables, n, cu=cu, max_q=2, want_lse=True)
        assert torch.isfinite(lse[:3]).all() and torch.all(lse[3:] == -math.inf)
    c = PagedKVCache(1, 8, 3, 64, 2, 64, 16, device=dev)
    step = c.step(torch.tensor([1, 0, 1], dtype=torch.int32, device=dev))
    x = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=dev)
    c.write(0, x, x, step)
    out, lse = c.attend(0, q[:3].contiguous(), step, want_lse=True)
    assert torch.all(out[:2] == 1) and not out[2].any() and torch.isfinite(lse[:2]).all() and torch.all(lse[2] == -math.inf)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("bad", [slice(0, 1), slice(0, 3), slice(2, None, 2), slice(0, None)])
def test_lse_beside_nan_values(dev, bad, sign, dtype):
    """The log-sum-exp is the keys' alone: value scales of NaN in some or all blocks make the outputs NaN and
    leave it as it is, for logits around 400 and around -400, in a short sequence and in one over many CTAs."""
    lens = [16, 40, 3000]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 2, 2, 64, 16, INT8, dtype, [1] * 3)
    kk = k.float()
    kk[..., 0] = 8.0
    slots = torch.cat([(tables[r].long()[:, None] * 16 + torch.arange(16, device=dev)).flatten()[:m] for r, m in enumerate(lens)])
    ops.cache_write(kk, v.float(), *pool, slots)
    k, v = (x.double() for x in ops.cache_read(*pool, slots, torch.float32))
    q[..., 0] = 400.0
    for r, m in enumerate(lens):
        pool[3][tables[r, :-(-m // 16)][bad].long()] = math.nan
    out, lse = ops.cache_attention(q, *pool, tables, n, scale=sign / 8, want_lse=True)
    b = 0
    for r, m in enumerate(lens):
        _, wl = ref.attention(q[r:r + 1].double(), k[b:b + m], v[b:b + m], sign / 8, True)
        mass = torch.einsum("mhd,nhd->mhn", q[r:r + 1].double().abs(), k[b:b + m].abs().repeat_interleave(2, 1)).amax(-1)
        assert torch.all((lse[r:r + 1].double() - wl).abs() <= 2.0 ** -20 * (1 + mass / 8) + 2.0 ** -23 * wl.abs())
        seen = tables[r, :-(-m // 16)][bad].numel() > 0
        assert torch.isnan(out[r]).all() if seen else torch.isfinite(out[r]).all()
        b += m


def test_attention_lengths_that_do_not_fit(dev):
    """Lengths below zero count as zero, lengths past the table as the table's; ``cu`` past the rows
    or falling leaves rows out, without a fault."""
    pool, tables, n, q, k, v = _attention_case(dev, [48, 30], 2, 2, 64, 16, E4M3, torch.bfloat16, [1] * 2)
    out, lse = ops.cache_attention(q, *pool, tables[:, :3].contiguous(), torch.tensor([10 ** 9, -4], dtype=torch.int32, device=dev),
                                   want_lse=True)
    _attention_check(out, lse, q, k, v, [48, 0], [1, 1], 64 ** -0.5, True)
    for cu in ([0, 5, 9], [0, 2, 1], [-3, 1, 2]):
        ops.cache_attention(q, *pool, tables, n, cu=torch.tensor(cu, dtype=torch.int32, device=dev), max_q=2)
    torch.cuda.synchronize()


def test_attention_long_offsets(dev):
    """Blocks beyond 2^31 bytes from the pool's start."""
    heads, dim, block = 8, 128, 128
    blocks = (1 << 31) // (heads * dim * block) + 40
    free, _ = torch.cuda.mem_get_info(dev)
    if free < 8 << 30:
        pytest.skip("needs 8 GB")
    pool = (torch.zeros(blocks, heads, block, dim, dtype=INT8, device=dev), torch.zeros(blocks, heads, block, dim, dtype=INT8, device=dev),
            torch.zeros(blocks, heads, device=dev), torch.zeros(blocks, heads, device=dev))
    ids = [blocks - 1, 0, blocks - 7]
    slots = torch.tensor([ids[i // block] * block + i % block for i in range(300)], device=dev)
    g = torch.Generator(device=dev).manual_seed(4)
    k, v = (torch.randn(300, heads, dim, generator=g, device=dev) for _ in range(2))
    ops.cache_write(k, v, *pool, slots)
    k, v = (x.double() for x in ops.cache_read(*pool, slots, torch.float32))
    q = torch.randn(1, 32, dim, generator=g, device=dev)
    out, lse = ops.cache_attention(q, *pool, torch.tensor([ids], dtype=torch.int32, device=dev),
                                   torch.tensor([300], dtype=torch.int32, device=dev), want_lse=True)
    _attention_check(out, lse, q, k, v, [300], [1], dim ** -0.5, True)


def test_attention_many_short_sequences(dev):
    """More units than the GPU has warps, several per warp."""
    lens = [(i * 37) % 200 for i in range(700)]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 4, 2, 64, 16, E4M3, torch.float16, [1] * len(lens))
    out, lse = ops.cache_attention(q, *pool, tables, n, want_lse=True)
    _attention_check(out, lse, q, k, v, lens, [1] * len(lens), 64 ** -0.5, True)


def test_attention_streams_and_graphs(dev):
    """Two streams at once, and two captured graphs replayed at once after their inputs changed, each
    give what a call alone gives."""
    cases = [_attention_case(dev, lens, 8, 4, 128, 16, E4M3, torch.bfloat16, [1] * len(lens), seed=i)
             for i, lens in enumerate(([3000, 17, 900], [5000, 40, 1]))]
    alone = [ops.cache_attention(c[3], *c[0], c[1], c[2]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(ops.cache_attention(c[3], *c[0], c[1], c[2]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    graphs, outs, qs = [], [], []
    for c in cases:
        q = c[3].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.cache_attention(q, *c[0], c[1], c[2]))
        graphs.append(g)
        qs.append(q)
    for r in range(10):
        for q, c in zip(qs, cases):
            q.copy_(c[3] * (1 if r % 2 else 0.5))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        if r % 2:
            assert all(torch.equal(a, b) for a, b in zip(outs, alone))


def test_launches_wait_for_what_comes_before(dev):
    """Kernels that may be placed early still wait: for a long kernel, a copy or a fill just before
    them on the stream, for another stream through an event, and eagerly as in a captured graph."""
    T, H, D = 4, 4, 64
    f, _ = rotary_frequencies(D, device=dev)
    pos = torch.arange(T, device=dev)
    src = torch.randn(T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(3))
    big = torch.randn(3000, 3000, device=dev)
    zero = torch.zeros(T, H, D, device=dev)
    want, _ = ops.rotary(src, None, pos, f)
    q = torch.empty_like(src)
    pool = _pool(dev, 4, H, 16, D, E4M3)
    slots = torch.arange(T, device=dev)

    def step():
        y = big @ big                                             # something long, then a small kernel
        q.copy_(src + 0 * y[0, 0])
        a, _ = ops.rotary(q, None, pos, f)
        q.zero_()                                                 # a fill and a copy of memory between the launches
        b, _ = ops.rotary(q, None, pos, f)
        q.copy_(src)
        ops.cache_write(q, q, *pool, slots)
        k, v = ops.cache_read(*pool, slots, torch.float32)
        return a, b, k, v

    r = ref.RefCache(H, 16, E4M3)
    r.write(src.double().cpu(), list(range(T)))
    held = r.read(list(range(T)), D).float()

    def check(got):
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], zero)
        assert torch.equal(got[2].cpu(), held) and torch.equal(got[3].cpu(), held)

    check(step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for t in got:
            t.fill_(7.0)
        graph.replay()
        check(got)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        q.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            y = big @ big
            q.copy_(src + 0 * y[0, 0])
            done = torch.cuda.Event()
            done.record()
        with torch.cuda.stream(b):
            b.wait_event(done)
            got, _ = ops.rotary(q, None, pos, f)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_attention_on_two_devices(dev):
    """The same call on each device of one process, whichever is current."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    lens = [300, 64]
    pool, tables, n, q, k, v = _attention_case(dev, lens, 2, 4, 128, 16, E4M3, torch.bfloat16, [1] * 2)
    want = ops.cache_attention(q, *pool, tables, n)
    other = torch.device("cuda", 1)
    got = ops.cache_attention(q.to(other), *(t.to(other) for t in pool), tables.to(other), n.to(other))
    assert got.device == other and torch.equal(got.to(dev), want)


def test_attention_refusals(dev):
    pool, tables, n, q, k, v = _attention_case(dev, [20, 30], 2, 2, 64, 16, E4M3, torch.bfloat16, [1] * 2)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    ok = dict(q=q, k_cache=pool[0], v_cache=pool[1], k_scale=pool[2], v_scale=pool[3], tables=tables, lens=n)
    for change, err in [(dict(q=q[:1]), ValueError), (dict(q=q[:, :3]), ValueError), (dict(q=q[..., :32]), ValueError),
                        (dict(q=q.double()), TypeError), (dict(tables=tables.long()), ValueError), (dict(tables=tables[:1]), ValueError),
                        (dict(lens=n.long()), ValueError), (dict(lens=n.cpu()), RuntimeError), (dict(cu=cu[:2]), ValueError),
                        (dict(cu=cu, max_q=0), RuntimeError), (dict(out=q.float()), ValueError), (dict(q=q.float().requires_grad_()), RuntimeError),
                        (dict(q=torch.zeros(2, 4, 65, dtype=torch.bfloat16, device=dev)[..., 1:]), RuntimeError),
                        (dict(cu=cu, max_q=1 << 20), RuntimeError)]:
        with pytest.raises(err):
            ops.cache_attention(**{**ok, **change})
    with pytest.raises(RuntimeError, match="geometry"):      # one row for all requests
        ops.cache_attention(**{**ok, "tables": tables[:1].expand(2, -1)})
    e = torch.empty(0, dtype=torch.int32, device=dev)
    assert ops.cache_attention(q[:0], *pool, tables[:0], e).shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,block", [(E4M3, 16), (INT8, 64)])
def test_evict_admit_and_decode(dev, fmt, block):
    """Prompts compressed by the hook enter the cache; then a loop of decode steps, one of them a
    prompt's end and another's beginning, against 64-bit attention over a 64-bit cache."""
    from submission_folder_b200.cluster import CircuitKVCluster, cli_cluster_kwargs
    from submission_folder_b200.synth import make_layer
    H, Hk, D, L = 32, 8, 128, 2
    inv, factor = rotary_frequencies(D, 10000.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=1024))
    cache = PagedKVCache(L, 40 * 16 // block * 2, 3, 700, Hk, D, block, fmt, inv_freq=inv, factor=factor, device=dev)
    held = [[None] * 3 for _ in range(L)]       # per layer and request: RefCache pair and slots
    layers = {}

    def admit(r, n, seed):
        kv = []
        for i in range(L):
            q, k, v = make_layer(n, seed=seed + i, window=32, planted=8, dtype="bf16")
            cl = CircuitKVCluster(**cli_cluster_kwargs(32, 128), distinct_kv_heads=bool(i))
            rep = [x.repeat_interleave(4, 0)[None].to(dev) for x in (k, v)]
            kv.append(cl.update_kv(rep[0], q[None].to(dev), rep[1], None, 4))
        step = cache.admit(r, kv, n)
        assert int(step.tables.granted[r]) == 128
        slots = step.tables.slots.tolist()
        assert slots == cache.slots(r, 128).tolist()
        for i, (k, v) in enumerate(kv):
            pair = [ref.RefCache(Hk, block, fmt), ref.RefCache(Hk, block, fmt)]
            for c, x in zip(pair, (k, v)):
                x = x[0, ::x.shape[1] // Hk].transpose(0, 1)
                c.write(x.double().cpu(), slots)
            held[i][r] = [pair, list(slots)]
        layers[r] = n

    admit(0, 700, 1)
    admit(2, 512, 11)
    g = torch.Generator(device=dev).manual_seed(6)
    for t in range(2 * block + 3 if block == 16 else 9):
        new = [1, 0, 1]
        if t == 4:
            new = [-1, 0, 2]
        if t > 4:
            new = [0, 1, 1]
        if t == 5:
            admit(1, 600, 21)
        step = cache.step(torch.tensor(new, dtype=torch.int32, device=dev), max_q=2)
        T = 6
        count = sum(max(x, 0) for x in new)
        pos = step.tables.positions.tolist()
        want_pos = []
        for r in range(3):
            for _ in range(max(new[r], 0)):
                want_pos.append(layers[r])
                layers[r] += 1
        assert pos[:count] == want_pos and step.tables.slots[count:].tolist() == [-1] * (T - count)
        for i in range(L):
            q, k, v = (torch.randn(T, h, D, generator=g, device=dev).bfloat16() for h in (H, Hk, Hk))
            out = cache.decode(i, q, k, v, step)
            assert not out[count:].any()
            qr, kr = ops.rotary(q, k, step.tables.positions, cache.inv_freq, factor=factor)
            a = 0
            for r in range(3):
                m = max(new[r], 0)
                if not m:
                    continue
                pair, slots = held[i][r]
                mine = step.tables.slots[a:a + m].tolist()
                for c, x in zip(pair, (kr, v)):
                    c.write(x[a:a + m].double().cpu(), mine)
                slots += mine
                kk, vv = (c.read(slots, D).to(dev) for c in pair)
                want, wl = ref.attention(qr[a:a + m].double(), kk, vv, D ** -0.5, True)
                _attention_check(out[a:a + m], wl.float(), qr[a:a + m], kk, vv, [len(slots)], [m], D ** -0.5, True)
                a += m
    k, v = cache.read(1, 2, len(held[1][2][1]), torch.float32)
    assert torch.equal(k[0].transpose(0, 1).double().cpu(), held[1][2][0][0].read(held[1][2][1], D))


def test_captured_decode_step(dev):
    """A whole decode step (tables, rotary, write, attention for two layers) captured once and
    replayed gives what eager steps give, across block borders."""
    H, Hk, D, L, R = 8, 2, 64, 2, 3
    inv, _ = rotary_frequencies(D)
    caches = [PagedKVCache(L, 64, R, 200, Hk, D, 16, inv_freq=inv, device=dev) for _ in range(2)]
    new = torch.tensor([1, 0, 1], dtype=torch.int32, device=dev)
    x = [torch.zeros(L, R, h, D, dtype=torch.bfloat16, device=dev) for h in (H, Hk, Hk)]

    def run(c):
        step = c.step(new)
        return torch.stack([c.decode(i, x[0][i], x[1][i], x[2][i], step) for i in range(L)])

    g = torch.Generator(device=dev).manual_seed(1)
    for t in x:
        t.normal_(generator=g)
    run(caches[1])                       # warm-up outside the capture, then the same start for both
    caches[1] = PagedKVCache(L, 64, R, 200, Hk, D, 16, inv_freq=inv, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = run(caches[1])
    for t in range(40):
        for a in x:
            a.normal_(generator=g)
        if t == 20:
            new.copy_(torch.tensor([1, 1, -1], dtype=torch.int32))
        if t == 21:
            new.copy_(torch.tensor([1, 1, 1], dtype=torch.int32))
        eager = run(caches[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, replayed), t
    for a, b in zip((caches[0].k, caches[0].lens, caches[0].tables, caches[0].free_count),
                    (caches[1].k, caches[1].lens, caches[1].tables, caches[1].free_count)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    del graph


def test_positions_of_a_row_that_is_used_again(dev):
    """A request ends after evictions; the next one of its row begins at position 0, and one that
    is refused leaves nothing behind."""
    c = PagedKVCache(1, 8, 2, 64, 2, 64, 16, device=dev)
    z = torch.zeros(1, 2, 20, 64, dtype=torch.bfloat16, device=dev)
    new = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    c.admit(0, [(z, z)], 500)
    c.admit(1, [(z, z)], 300)
    assert c.step(new(1, 1)).tables.positions.tolist() == [500, 300]
    c.step(new(-1, 0))
    assert c.step(new(1, 1)).tables.positions.tolist() == [0, 301]
    c.step(new(-1, 1))
    big = z.repeat(1, 1, 4, 1)
    step = c.admit(0, [(big, big)], 900)                        # 80 tokens, 64 fit the row
    assert int(step.tables.granted[0]) == 0
    assert c.step(new(2, 1), total=3).tables.positions.tolist() == [0, 1, 303]
    with pytest.raises(ValueError):
        c.read(0, 0, 65)
    assert c.read(0, 0, 64)[0].shape == (1, 2, 64, 64) and c.read(0, 1, 0)[0].shape == (1, 2, 0, 64)


@pytest.mark.parametrize("captured", [False, True])
def test_refused_requests_attend_to_nothing(dev, captured):
    """A request that gets no room, for lack of blocks or of places in its row, gives zeros from ``decode``
    while it keeps its length; the others, one refused earlier among them, go on as if it had not asked."""
    D, R = 64, 4
    new = torch.zeros(R, dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    x = [torch.zeros(2 * R, h, D, dtype=torch.bfloat16, device=dev) for h in (4, 2, 2)]

    def run(c):
        step = c.step(new, max_q=2)
        return c.decode(0, *x, step), step

    def fresh():
        c = PagedKVCache(1, 7, R, 48, 2, D, 16, device=dev)
        for r, n in enumerate((30, 46, 16, 16)):
            z = torch.randn(1, 2, n, D, generator=torch.Generator().manual_seed(r)).bfloat16().to(dev)
            assert int(c.admit(r, [(z, z)], n).tables.granted[r]) == n
        return c

    c, want = fresh(), fresh()
    # (asked, granted): 0 blocks left; then one comes back with request 2's end
    steps = [((1, 2, 1, 2), (1, 2, 0, 0)), ((1, 1, 0, 1), (1, 0, 0, 0)), ((0, 0, -1, 1), (0, 0, 0, 1)), ((2, 1, 1, 2), (0, 0, 0, 2))]
    if captured:
        run(fresh())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, step = run(c)
    for asked, granted in steps:
        for t in x:
            t.normal_(generator=g)
        new.copy_(torch.tensor(asked, dtype=torch.int32))
        if captured:
            graph.replay()
        else:
            got, step = run(c)
        assert step.tables.granted.tolist() == list(granted)
        a = 0
        for r in range(R):
            m = max(asked[r], 0)
            if m and not granted[r]:
                assert not got[a:a + m].any()
            a += m
        assert not got[a:].any()
        # the same step without those that are refused
        keep = [i for i, r in enumerate(r for r in range(R) for _ in range(max(asked[r], 0))) if granted[r]]
        y = [torch.cat([t[keep], t[:2 * R - len(keep)]]) for t in x]
        alone = want.step(torch.tensor([n if n < 0 else m for n, m in zip(asked, granted)], dtype=torch.int32, device=dev), max_q=2)
        assert torch.equal(want.decode(0, *y, alone)[:len(keep)], got[keep])
        assert torch.equal(want.lens, c.lens) and torch.equal(want.free_count, c.free_count)
    if captured:
        del graph


def test_rows_that_overlap_are_refused(dev):
    pool = _pool(dev, 4, 2, 16, 64, E4M3)
    x, slots = torch.ones(3, 2, 64, device=dev), torch.arange(3, device=dev)
    f, _ = rotary_frequencies(64, device=dev)
    t, n = torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    same = torch.empty(1, 2, 64, device=dev).expand(3, 2, 64)
    flat = pool[0].view(torch.uint8)[:1].expand(4, 2, 16, 64).view(E4M3)
    for call in (lambda: ops.rotary(x, None, slots, f, out=(same, None)), lambda: ops.rotary(x, x, slots, f, out=(x.clone(), same)),
                 lambda: ops.cache_write(x, x, flat, *pool[1:], slots), lambda: ops.cache_write(x, x, pool[0], *pool[:1], *pool[2:], slots),
                 lambda: ops.cache_attention(x, *pool, t, n, out=same)):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    with pytest.raises(ValueError, match="out"):
        ops.rotary(x, x, slots, f, out=(None, x.clone()))
    ops.cache_read(flat, flat, *pool[2:], slots)               # reading them is fine
    ops.rotary(same, same, slots, f)


def test_tangents_are_refused(dev):
    """Forward-mode derivatives would be dropped quietly."""
    import torch.autograd.forward_ad as fw
    pool = _pool(dev, 4, 2, 16, 64, E4M3)
    x, slots = torch.ones(3, 2, 64, device=dev), torch.arange(3, device=dev)
    f, _ = rotary_frequencies(64, device=dev)
    t, n = torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    with fw.dual_level():
        d = fw.make_dual(x, x)
        for call in (lambda y: ops.rotary(y, None, slots, f), lambda y: ops.rotary(x, y, slots, f),
                     lambda y: ops.cache_write(y, x, *pool, slots), lambda y: ops.cache_write(x, y, *pool, slots),
                     lambda y: ops.cache_attention(y, *pool, t, n), lambda y: ops.cache_attention(x, *pool, t, n, out=y)):
            with pytest.raises(RuntimeError, match="tangents"):
                call(d)
            call(d.detach().clone())


def test_written_tensors_change_their_version(dev):
    """Autograd sees that a saved tensor was overwritten; what is only read keeps its version."""
    i32 = dict(dtype=torch.int32, device=dev)
    pool = _pool(dev, 4, 2, 16, 64, E4M3)
    x, slots = torch.ones(3, 2, 64, device=dev), torch.arange(3, device=dev)
    f, _ = rotary_frequencies(64, device=dev)
    a = [torch.zeros(3, **i32), torch.ones(3, **i32), torch.zeros(3, 2, **i32), torch.arange(4, **i32), torch.tensor([4], **i32)]
    out = torch.empty_like(x), torch.empty_like(x)

    def changed(ts, call):
        before = [t._version for t in ts]
        call()
        return [t._version > b for t, b in zip(ts, before)]

    assert changed(a, lambda: ops.block_tables(*a, 16, 3)) == [True, False, True, True, True]
    apart = torch.empty(3, **i32), torch.empty(1, **i32)
    assert changed([a[0], a[4], *apart], lambda: ops.block_tables(*a, 16, 3, lens_out=apart[0], free_count_out=apart[1])) == [False, False, True, True]
    assert changed([x, *out], lambda: ops.rotary(x, x.clone(), slots, f, out=out)) == [False, True, True]
    assert changed([x, *pool], lambda: ops.cache_write(x, x, *pool, slots)) == [False] + [True] * 4
    assert changed(pool, lambda: ops.cache_read(*pool, slots)) == [False] * 4
    assert changed([x, out[0], *pool], lambda: ops.cache_attention(x, *pool, a[2], a[1], out=out[0])) == [False, True] + [False] * 4
    w = torch.ones(3, 2, 64, device=dev, requires_grad=True)
    y = w * out[0]
    ops.cache_attention(x, *pool, a[2], a[1], out=out[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        z = torch.empty_like(x)
    ops.cache_attention(x, *pool, a[2], a[1], out=z)          # tensors of inference mode have no version


def test_a_refused_prompt_takes_nothing(dev):
    """Layers that cannot be written are refused before any block is taken: the cache is as it was."""
    c = PagedKVCache(2, 8, 2, 64, 2, 64, 16, device=dev)
    z = torch.zeros(1, 2, 20, 64, dtype=torch.bfloat16, device=dev)
    c.admit(1, [(z, z)] * 2, 30)
    state = [t.clone() for t in (c.lens, c.tables, c.free_list, c.free_count, c.shift)]
    odd = torch.zeros(1, 2, 20, 65, dtype=torch.bfloat16, device=dev)[..., 1:]
    for bad, err in [(z.double(), TypeError), (z.cpu(), RuntimeError), (torch.cat([z, z], -1), ValueError),
                     (z.clone().requires_grad_(), RuntimeError), (odd, ValueError), (z.transpose(2, 3).contiguous().transpose(2, 3), ValueError)]:
        for layers in ([(bad, bad)] * 2, [(z, z), (bad, bad)], [(z, z), (z, bad)]):
            with pytest.raises((err, ValueError)):
                c.admit(0, layers, 40)
            assert all(torch.equal(a, b) for a, b in zip(state, (c.lens, c.tables, c.free_list, c.free_count, c.shift)))
    assert c.admit(0, [(z, z)] * 2, 40).tables.granted.tolist() == [20, 0]


def test_admission_to_a_busy_row_changes_nothing(dev):
    """A prompt for a row that holds a request: the request keeps its tokens, blocks and positions."""
    c = PagedKVCache(1, 8, 2, 64, 2, 64, 16, device=dev)
    z = [torch.randn(1, 2, n, 64, generator=torch.Generator().manual_seed(n)).bfloat16().to(dev) for n in (20, 7, 0)]
    c.admit(0, [(z[0], z[0])], 500)
    held = [t.clone() for t in (c.lens, c.tables, c.free_list, c.free_count, c.shift, c.k.view(torch.uint8), c.k_scale)]
    for x in z[1:]:
        step = c.admit(0, [(x, x)], 90)
        assert int(step.tables.granted[0]) == 0 and step.tables.slots.tolist() == [-1] * x.shape[2]
        now = (c.lens, c.tables, c.free_list, c.free_count, c.shift, c.k.view(torch.uint8), c.k_scale)
        assert all(torch.equal(a, b) for a, b in zip(held, now))
    assert c.step(torch.tensor([1, 0], dtype=torch.int32, device=dev)).tables.positions.tolist() == [500, 0]


def test_a_refused_prompt_of_more_than_max_q_tokens(dev):
    """Zeros, as for any request that did not fit, also where its rows are more than the step's ``max_q``."""
    c = PagedKVCache(1, 4, 2, 64, 2, 64, 16, device=dev)
    step = c.step(torch.tensor([1, 70], dtype=torch.int32, device=dev), total=9)
    x = torch.ones(9, 2, 64, dtype=torch.bfloat16, device=dev)
    out = c.decode(0, x, x, x, step)
    assert step.tables.granted.tolist() == [1, 0] and torch.all(out[0] == 1) and not out[1:].any()


def test_paged_cache_class_refusals(dev):
    c = PagedKVCache(1, 8, 2, 64, 2, 64, 16, device=dev)
    z = torch.zeros(1, 2, 20, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        c.admit(0, [], 20)
    with pytest.raises(ValueError):
        c.admit(0, [(z, z[:, :, :5])], 20)
    with pytest.raises(ValueError):
        c.admit(0, [(z[:, :1], z[:, :1])], 20)
    with pytest.raises(ValueError):
        c.admit(0, [(z, z)], 19)
    step = c.admit(0, [(z.repeat(1, 1, 4, 1), z.repeat(1, 1, 4, 1))], 80)      # 80 tokens, 64 fit the row
    assert int(step.tables.granted[0]) == 0 and int(c.lens[0]) == 0 and int(c.free_count) == 8
