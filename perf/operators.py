"""The operators of a paged 8-bit decode cache, as measured work: their cases, their plain forms and their calls.

After a prefill layer's eviction the kept keys and values go into blocks of a pool, held in 8 bits with one scale for
each (block, KV head).  A decode step then needs four things, and a fifth when a cache is compressed again:

* tables     block tables, slots and positions of the step's tokens from the requests' lengths
* rotary     rotary positions of the new queries and keys (and the gradient, which is the inverse rotation)
* write      the new keys and values into their blocks
* read       tokens of the pool back as numbers, for another round of scoring
* attention  of the new queries over the blocks

``own`` is set from outside: false computes the plain forms below, true calls the library.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    heads = {"q_heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # one decode step of a batch of 16: a token each, now and then a new block
        {"name": "tables_decode_16", "kind": "tables", "requests": 16, "block": 16, "longest": 3277, "mix": "decode"},
        # a busy scheduler step: 1024 rows that decode, idle, end, or bring a prompt's kept tokens
        {"name": "tables_mixed_1024", "kind": "tables", "requests": 1024, "block": 32, "longest": 4096, "mix": "mixed"},
        # the decode step's queries and keys, all at far positions of their own
        {"name": "rotary_decode_16", "kind": "rotary", "tokens": 16, "dtype": "bf16", "rotary_dim": 128,
         "interleaved": False, "inverse": False, "scaling": "none", **heads},
        # a 32k prompt with positions scaled for a long context
        {"name": "rotary_prompt_32k", "kind": "rotary", "tokens": 32768, "dtype": "bf16", "rotary_dim": 128,
         "interleaved": False, "inverse": False, "scaling": "ramp", **heads},
        # gradients with respect to the unrotated queries and keys: interleaved pairs, half of the head, odd length
        {"name": "rotary_grad_8191", "kind": "rotary", "tokens": 8191, "dtype": "fp32", "rotary_dim": 64,
         "interleaved": True, "inverse": True, "scaling": "linear", **heads},
        # one new token for each of 16 sequences, into blocks that hold others already
        {"name": "write_append_16", "kind": "write", "sequences": 16, "longest": 3277, "tokens_each": 1, "block": 16,
         "format": "e4m3", "dtype": "bf16", "kv_heads": 8, "dim": 128},
        # the kept tokens of 16 ragged prompts (a tenth of 2048..32768) into fresh blocks
        {"name": "write_prompts_16", "kind": "write", "sequences": 16, "longest": 3277, "tokens_each": 0, "block": 32,
         "format": "e4m3", "dtype": "bf16", "kv_heads": 8, "dim": 128},
        # a whole 131072-token context written in int8 and read back for another round of scoring
        {"name": "write_read_131072", "kind": "write_read", "sequences": 1, "longest": 131072, "tokens_each": 0,
         "block": 64, "format": "int8", "dtype": "fp16", "kv_heads": 8, "dim": 128},
        # one sequence with the smallest budget: latency
        {"name": "attention_1x512", "kind": "attention", "sequences": 1, "shortest": 512, "longest": 512, "queries": 1,
         "block": 16, "format": "e4m3", "dtype": "bf16", **heads},
        # the batched serving sweep: 16 ragged sequences, a tenth of 2048..32768 kept
        {"name": "attention_16_ragged", "kind": "attention", "sequences": 16, "shortest": 205, "longest": 3277,
         "queries": 1, "block": 32, "format": "e4m3", "dtype": "bf16", **heads},
        # four tokens to verify against one uncompressed 131072-token context
        {"name": "attention_verify_131072", "kind": "attention", "sequences": 1, "shortest": 131072, "longest": 131072,
         "queries": 4, "block": 64, "format": "int8", "dtype": "fp32", **heads},
        # a large batch of long uncompressed contexts: bandwidth
        {"name": "attention_32x32k", "kind": "attention", "sequences": 32, "shortest": 2048, "longest": 32768,
         "queries": 1, "block": 64, "format": "e4m3", "dtype": "bf16", **heads},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rotary", "rotary", "write", "write_read", "attention", "attention", "attention"])
    if kind == "tables":
        return {"kind": kind, "requests": _log_int(rng, 1, 1024), "block": rng.choice([16, 32, 64, 128]),
                "longest": _log_int(rng, 64, 4096), "mix": rng.choice(["decode", "mixed"])}
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 128])
    if kind == "rotary":
        return {"kind": kind, "tokens": _log_int(rng, 1, 16384), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "rotary_dim": rng.choice([dim, dim, dim // 2, dim // 4, dim - 6]), "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.3, "scaling": rng.choice(["none", "linear", "ramp"]),
                "q_heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim}
    block = rng.choice([16, 32, 64, 128])
    fmt, dt = rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "fp16", "fp32"])
    if kind in ("write", "write_read"):
        fresh = rng.random() < 0.5
        seqs = rng.randint(1, 16) if fresh else _log_int(rng, 1, 256)
        return {"kind": kind, "sequences": seqs, "longest": _log_int(rng, 17, 4096),
                "tokens_each": 0 if fresh else rng.randint(1, 5), "block": block, "format": fmt, "dtype": dt,
                "kv_heads": kv, "dim": dim}
    seqs = _log_int(rng, 1, 64)
    longest = _log_int(rng, 1, max(1, min(131072, 500000 // seqs)))
    return {"kind": kind, "sequences": seqs, "shortest": max(1, longest // rng.choice([1, 3, 10])), "longest": longest,
            "queries": rng.choice([1, 1, 1, 2, 3, 5]), "block": block, "format": fmt, "dtype": dt,
            "q_heads": kv * rng.choice([1, 2, 4, 4, 7, 8]), "kv_heads": kv, "dim": dim}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _shape_rng(case):
    """Lengths go by the case alone, so that every seed has outputs of the same sizes."""
    return np.random.default_rng([case.get("requests", 0) + case.get("sequences", 0), case["longest"], case["block"]])


def _lengths(case):
    """Lengths of the sequences, spread evenly over the case's range; the longest one is there."""
    rng = _shape_rng(case)
    lo, hi = case.get("shortest", max(1, case["longest"] // 16)), case["longest"]
    lens = rng.integers(lo, hi + 1, case["sequences"])
    lens[rng.integers(case["sequences"])] = hi
    return lens


def _pool(lens, block, rng):
    """A block table for each sequence, over a shuffled pool with a few spare blocks."""
    need = -(-lens // block)
    order = rng.permutation(int(need.sum()) + 3)
    tables = np.zeros((len(lens), int(need.max()) + 1), np.int32)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = order[at:at + n]
        at += n
    return tables, len(order)


def _frequencies(case):
    """Radians per position of each pair, and the factor on cosine and sine."""
    d = case["rotary_dim"]
    i = np.arange(0, d, 2, dtype=np.float64) / d
    f = 10000.0 ** -i
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "ramp":
        # whole turns over 8192 positions: fast pairs stay, slow pairs are stretched by 16, a ramp between
        turns = 8192 * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * (keep + (1 - keep) / 16.0), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _scale(amax, fmt):
    """The smallest power of two (2^-126 at least) with amax / scale at most the format's largest value: 448 or 127."""
    m, x = torch.frexp(amax)   # amax = m 2^x, m in [0.5, 1); 448 = 0.875 2^9, 127 = 0.9921875 2^7
    e = x - 9 + (m > 0.875).int() if fmt == "e4m3" else x - 7 + (m > 0.9921875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, fmt):
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else x.round().to(torch.int8)


def _filled(blocks, case, gen):
    """A pool of ``blocks`` blocks of normal values, each (block, head) with its scale."""
    shape = (case["kv_heads"], case["block"], case["dim"])
    codes = torch.empty(blocks, *shape, dtype=CODES[case["format"]], device=DEV)
    scale = torch.empty(blocks, case["kv_heads"], dtype=torch.float32, device=DEV)
    step = max(1, (1 << 26) // math.prod(shape))
    for a in range(0, blocks, step):
        x = torch.randn(min(step, blocks - a), *shape, generator=gen, device=DEV)
        s = _scale(x.abs().amax((2, 3)), case["format"])
        scale[a:a + step] = s
        codes[a:a + step] = _codes(x / s[:, :, None, None], case["format"])
    return codes, scale


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    kind = case["kind"]
    if kind == "tables":
        R, block, sizes = case["requests"], case["block"], _shape_rng(case)
        lens = sizes.integers(1, case["longest"] + 1, R)
        new = np.ones(R, np.int64)
        if case["mix"] == "mixed":
            what = sizes.random(R)
            new[what < 0.3] = 0                              # idle
            new[what < 0.2] = -1                             # ended: the blocks go back
            prompt = what > 0.7
            lens[prompt] = 0
            new[prompt] = sizes.integers(1, case["longest"] + 1, int(prompt.sum()))
        total = int(new.clip(0).sum()) + int(sizes.integers(0, 4))   # a padded batch has tokens of no request
        width = -(-(case["longest"] * 2) // block)
        tables, used = _pool(lens, block, rng)
        full = np.zeros((R, width), np.int32)
        full[:, :min(width, tables.shape[1])] = tables[:, :width]
        spare = int((-(-(lens + new.clip(0)) // block)).sum() - (-(-lens // block)).sum()) + 2
        free = np.full(used + spare, -1, np.int32)
        free[:spare] = used + rng.permutation(spare)
        st.update(lens=_dev(lens.astype(np.int32)), new=_dev(new.astype(np.int32)), tables=_dev(full),
                  shift=_dev(rng.integers(0, 131072, R).astype(np.int32)), free=_dev(free),
                  count=_dev(np.array([spare], np.int32)), total=total,
                  lens_out=torch.empty(R, dtype=torch.int32, device=DEV),
                  count_out=torch.empty(1, dtype=torch.int32, device=DEV))
        return st
    if kind == "rotary":
        T, D, dt = case["tokens"], case["dim"], DTYPES[case["dtype"]]
        f, factor = _frequencies(case)
        st.update(q=torch.randn(T, case["q_heads"], D, generator=gen, device=DEV).to(dt),
                  k=torch.randn(T, case["kv_heads"], D, generator=gen, device=DEV).to(dt),
                  positions=_dev(rng.integers(0, 131072, T) if T <= 256 else np.arange(T) + rng.integers(0, 98304)),
                  inv_freq=_dev(f), factor=factor)
        return st
    lens = _lengths(case)
    tables, blocks = _pool(lens, case["block"], rng)
    if kind in ("write", "write_read"):
        st["k_cache"], st["k_scale"] = _filled(blocks, case, gen)
        st["v_cache"], st["v_scale"] = _filled(blocks, case, gen)
        n = case["tokens_each"]
        slots = []
        for r, length in enumerate(lens):
            pos = np.arange(0 if n == 0 else max(0, length - n), length)   # 0: the whole sequence; else its last tokens
            slots.append(tables[r, pos // case["block"]].astype(np.int64) * case["block"] + pos % case["block"])
        st["slots"] = _dev(np.concatenate(slots))
        T, dt = st["slots"].numel(), DTYPES[case["dtype"]]
        # keys have a few strong channels
        loud = 1.0 + 7.0 * (torch.rand(case["kv_heads"], case["dim"], generator=gen, device=DEV) < 0.03)
        st["k"] = (torch.randn(T, case["kv_heads"], case["dim"], generator=gen, device=DEV) * loud).to(dt)
        st["v"] = torch.randn(T, case["kv_heads"], case["dim"], generator=gen, device=DEV).to(dt)
        return st
    st["k_cache"], st["k_scale"] = _filled(blocks, case, gen)
    st["v_cache"], st["v_scale"] = _filled(blocks, case, gen)
    T = case["sequences"] * case["queries"]
    q = 1.5 * torch.randn(T, case["q_heads"], case["dim"], generator=gen, device=DEV)   # some keys stand out
    st.update(q=q.to(DTYPES[case["dtype"]]), tables=_dev(tables), lens=_dev(lens.astype(np.int32)),
              cu=_dev(np.arange(0, T + 1, case["queries"], dtype=np.int32)), scale=case["dim"] ** -0.5)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        return _run_own(st, case, kind)
    if kind == "tables":
        return _plain_tables(st, case["block"])
    if kind == "rotary":
        return {n: _plain_rotary(st[n], st, case) for n in ("q", "k")}
    if kind == "write":
        _plain_write(st, case)
        return {n: st[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if kind == "write_read":
        _plain_write(st, case)
        return {n: _plain_read(st, n, case) for n in ("k", "v")}
    return _plain_attention(st, case)


def _run_own(st, case, kind):
    from submission_folder_b200 import ops
    if kind == "tables":
        p = ops.block_tables(st["lens"], st["new"], st["tables"], st["free"], st["count"], case["block"], st["total"],
                             shift=st["shift"], lens_out=st["lens_out"], free_count_out=st["count_out"])
        return {"lens": p.lens, "tables": st["tables"], "free": st["free"], "count": p.free_count, "cu": p.cu,
                "slots": p.slots, "positions": p.positions, "granted": p.granted}
    if kind == "rotary":
        q, k = ops.rotary(st["q"], st["k"], st["positions"], st["inv_freq"], interleaved=case["interleaved"],
                          factor=st["factor"], inverse=case["inverse"])
        return {"q": q, "k": k}
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if kind in ("write", "write_read"):
        ops.cache_write(st["k"], st["v"], *cache, st["slots"])
        if kind == "write":
            return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache))
        k, v = ops.cache_read(*cache, st["slots"], DTYPES[case["dtype"]])
        return {"k": k, "v": v}
    out, lse = ops.cache_attention(st["q"], *cache, st["tables"], st["lens"], cu=st["cu"], max_q=case["queries"],
                                   scale=st["scale"], want_lse=True)
    return {"out": out, "lse": lse}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_tables(st, block):
    lens, new, tables, free, shift = (st[n].long() for n in ("lens", "new", "tables", "free", "shift"))
    count, T, width = st["count"].long(), st["total"], tables.shape[1]
    held = (lens + block - 1) // block
    back = torch.where(new < 0, held, torch.zeros_like(held))
    ask = new.clamp(min=0)
    # the blocks of ended requests go on top of the free list, in the requests' order
    col = torch.arange(width, device=DEV)
    at = count + (back.cumsum(0) - back)[:, None] + col
    at = torch.where(col < back[:, None], at, torch.full_like(at, free.numel()))
    free = torch.cat([free, free.new_zeros(1)]).scatter(0, at.reshape(-1), tables.reshape(-1))[:-1]
    have = count + back.sum()
    # fresh blocks are taken from the top, in the requests' order
    need = (lens + ask + block - 1) // block - held
    fits = held + need <= width
    need = torch.where(fits & (new >= 0), need, torch.zeros_like(need))
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= have))
    granted = torch.where(ok, ask, torch.zeros_like(ask))
    need = torch.where(ok, need, torch.zeros_like(need))
    nth = (upto - need)[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    tables = torch.where(fresh, free[(have - 1 - nth).clamp(0, free.numel() - 1)], tables)
    lens_out = torch.where(new < 0, torch.zeros_like(lens), lens + granted)
    cu = torch.cat([ask.new_zeros(1), ask.cumsum(0)])
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(cu, t, right=True) - 1
    real = t < cu[-1]
    r = r.clamp(0, lens.numel() - 1)
    pos = lens[r] + t - cu[r]
    slots = tables[r, (pos // block).clamp(max=width - 1)] * block + pos % block
    slots = torch.where(real & (granted[r] > 0), slots, torch.full_like(slots, -1))
    positions = torch.where(real, pos + shift[r], torch.zeros_like(pos))
    i32 = torch.int32
    return {"lens": lens_out.to(i32), "tables": tables.to(i32), "free": free.to(i32),
            "count": (have - need.sum()).to(i32), "cu": cu.to(i32), "slots": slots, "positions": positions,
            "granted": granted.to(i32)}


def _plain_rotary(x, st, case):
    d = case["rotary_dim"]
    angle = st["positions"].double()[:, None] * st["inv_freq"]
    cos, sin = (angle.cos() * st["factor"]).float()[:, None], (angle.sin() * st["factor"]).float()[:, None]
    if case["inverse"]:
        sin = -sin
    y = x.float()
    a, b = (y[..., :d:2], y[..., 1:d:2]) if case["interleaved"] else (y[..., :d // 2], y[..., d // 2:d])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if case["interleaved"] else torch.cat([u, w], -1)
    return torch.cat([turned, y[..., d:]], -1).to(x.dtype)


def _plain_write(st, case):
    block, fmt = case["block"], case["format"]
    b, off = st["slots"] // block, st["slots"] % block
    blocks = st["k_cache"].shape[0]
    # a write of a block's first token begins the block anew; another one keeps what the block holds
    anew = _began(b, off, blocks)
    for name in ("k", "v"):
        codes, scale, x = st[name + "_cache"], st[name + "_scale"], st[name].float()
        top = torch.zeros(blocks, case["kv_heads"], device=DEV)
        top = top.scatter_reduce(0, b[:, None].expand(-1, case["kv_heads"]), x.abs().amax(-1), "amax")
        touched = torch.zeros(blocks, dtype=torch.bool, device=DEV).index_fill(0, b, True)
        new = _scale(top, fmt)
        new = torch.where(anew[:, None], new, torch.maximum(new, scale))
        new = torch.where(touched[:, None], new, scale)
        ratio = torch.where(anew[:, None], torch.ones_like(new), scale / new)   # 1 where nothing grows
        codes.copy_(_codes(codes.float() * ratio[:, :, None, None], fmt))
        codes.view(torch.uint8)[b, :, off] = _codes(x / new[b][..., None], fmt).view(torch.uint8)
        scale.copy_(new)


def _began(b, off, blocks):
    first = torch.where(off == 0, b, torch.full_like(b, blocks))
    return torch.zeros(blocks + 1, dtype=torch.bool, device=DEV).index_fill(0, first, True)[:blocks]


def _plain_read(st, name, case):
    b, off = st["slots"] // case["block"], st["slots"] % case["block"]
    codes = st[name + "_cache"].view(torch.uint8)[b, :, off].view(CODES[case["format"]])
    return (codes.float() * st[name + "_scale"][b][..., None]).to(DTYPES[case["dtype"]])


def _plain_attention(st, case):
    block, nq, R = case["block"], case["queries"], case["sequences"]
    H, G, D = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"]
    lens = st["lens"].long()
    width = -(-case["longest"] // block)
    tables = st["tables"][:, :width].long()
    q = st["q"].float().view(R, nq, H, G, D).permute(0, 2, 1, 3, 4).reshape(R, H, nq * G, D)

    def rows(name):
        codes = st[name + "_cache"].view(torch.uint8)[tables].view(CODES[case["format"]])   # [R, width, H, block, D]
        x = codes.float() * st[name + "_scale"][tables][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(R, H, width * block, D)

    s = torch.matmul(q, rows("k").transpose(-1, -2)) * st["scale"]
    # query i of nq sees the sequence up to its own place: lens - nq + i + 1 tokens
    sees = lens[:, None] - nq + 1 + torch.arange(nq, device=DEV)
    sees = sees.repeat_interleave(G, 1)[:, None, :, None]
    s = s.masked_fill(torch.arange(width * block, device=DEV) >= sees, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = (s - m).exp()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows("v")) / torch.where(z > 0, z, torch.ones_like(z))
    lse = (z.log() + m).squeeze(-1)

    def back(x):   # [R, H, nq * G, ...] -> [T, H * G, ...]
        x = x.reshape(R, H, nq, G, *x.shape[3:])
        return x.transpose(1, 2).reshape(R * nq, H * G, *x.shape[4:])

    return {"out": back(o).to(st["q"].dtype), "lse": back(lse)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}.get(case.get("dtype"), 0)
    kind = case["kind"]
    if kind == "tables":
        R, mean = case["requests"], case["longest"] / 2
        if case["mix"] == "decode":
            return {"bytes": R * (4 * 6 + 16 + 4 / case["block"] * 2), "flops": 0}
        tokens = R * 0.3 * mean + R * 0.4
        moved = 0.5 * R * mean / case["block"]
        return {"bytes": R * 24 + tokens * 16 + moved * 8, "flops": 0}
    if kind == "rotary":
        heads = case["q_heads"] + case["kv_heads"]
        n = case["tokens"] * heads
        return {"bytes": 2 * n * case["dim"] * size + case["tokens"] * 8, "flops": 3 * n * case["rotary_dim"]}
    if kind in ("write", "write_read"):
        mean = case["longest"] if case["sequences"] == 1 else case["longest"] * 17 / 32
        each = case["tokens_each"] or mean
        n = case["sequences"] * each * case["kv_heads"]
        moved = 2 * n * case["dim"] * (size + 1)
        if kind == "write_read":
            moved += 2 * n * case["dim"] * (size + 1)
        return {"bytes": moved + case["sequences"] * each * 8, "flops": 0}
    mean = case["longest"] if case["sequences"] == 1 else (case["shortest"] + case["longest"]) / 2
    keys = case["sequences"] * mean
    rows = case["sequences"] * case["queries"] * case["q_heads"]
    cache = 2 * keys * case["kv_heads"] * (case["dim"] + 4 / case["block"])
    return {"bytes": cache + 2 * rows * case["dim"] * size + rows * 4,
            "flops": 4 * keys * case["queries"] * case["q_heads"] * case["dim"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":
        return _exact_tables(st, case["block"])
    if kind == "rotary":
        return {n: _exact_rotary(st[n], st, case) for n in ("q", "k")}
    if kind in ("write", "write_read"):
        return _exact_write(st, case, kind == "write_read")
    return _exact_attention(st, case)


def _exact_tables(st, block):
    lens, new, tables, free, shift = (st[n].cpu().numpy().astype(np.int64).copy()
                                      for n in ("lens", "new", "tables", "free", "shift"))
    count, T = int(st["count"]), st["total"]
    R = len(lens)
    for r in range(R):
        if new[r] < 0:
            n = -(-int(lens[r]) // block)
            free[count:count + n] = tables[r, :n]
            count += n
    cu, slots, positions = np.zeros(R + 1, np.int64), np.full(T, -1, np.int64), np.zeros(T, np.int64)
    granted, short = np.zeros(R, np.int64), False
    out = lens.copy()
    for r in range(R):
        n = max(int(new[r]), 0)
        cu[r + 1] = cu[r] + n
        if new[r] < 0:
            out[r] = 0
            continue
        pos = lens[r] + np.arange(n)
        positions[cu[r]:cu[r + 1]] = pos + shift[r]
        have, want = -(-int(lens[r]) // block), -(-int(lens[r] + n) // block)
        if want > tables.shape[1]:
            continue
        if want > have:
            short = short or want - have > count
            if short:
                continue
            for c in range(have, want):
                count -= 1
                tables[r, c] = free[count]
        granted[r], out[r] = n, lens[r] + n
        slots[cu[r]:cu[r + 1]] = tables[r, pos // block] * block + pos % block
    i32 = np.int32
    return {"lens": out.astype(i32), "tables": tables.astype(i32), "free": free.astype(i32),
            "count": np.array([count], i32), "cu": cu.astype(i32), "slots": slots, "positions": positions,
            "granted": granted.astype(i32)}


def _exact_rotary(x, st, case):
    d = case["rotary_dim"]
    angle = torch.outer(st["positions"].double(), st["inv_freq"].double())
    turn = torch.polar(torch.full_like(angle, st["factor"]), -angle if case["inverse"] else angle)[:, None]
    y = x.double()
    head = y[..., :d]
    pairs = head.unflatten(-1, (d // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y[..., :d] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return y


def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round(x, fmt):
    """float64 values to the nearest value of the format, ties to even."""
    if fmt == "int8":
        return x.round()
    _, e = torch.frexp(x)                                    # |x| < 2^e: 4 significant bits, spacing 2^(e - 4)
    step = _two_to((e - 4).clamp(min=-9))
    return (x / step).round() * step


def _exact_write(st, case, values):
    block, fmt = case["block"], case["format"]
    largest = 448.0 if fmt == "e4m3" else 127.0
    slots = st["slots"].cpu().numpy()
    b = slots // block
    starts = np.flatnonzero(np.r_[True, b[1:] != b[:-1]])
    ends = np.r_[starts[1:], len(b)]
    if len(starts) > 12000:
        return None
    got = {}
    for name in ("k", "v"):
        codes, scale, x = st[name + "_cache"].double(), st[name + "_scale"].double(), st[name].double()
        for a, z in zip(starts.tolist(), ends.tolist()):
            n, first = int(b[a]), int(slots[a] % block)
            rows = x[a:z].transpose(0, 1)                    # [heads, tokens, dim]; consecutive offsets of one block
            want = _two_to(torch.ceil(torch.log2(rows.abs().amax((1, 2)) / largest)).clamp(min=-126))
            if first:
                want = torch.maximum(want, scale[n])
                codes[n] = _exact_round(codes[n] * (scale[n] / want)[:, None, None], fmt)
            codes[n, :, first:first + z - a] = _exact_round(rows / want[:, None, None], fmt)
            scale[n] = want
        if values:
            at = st["slots"]
            got[name] = codes[at // block, :, at % block] * scale[at // block][..., None]
        else:
            got[name + "_cache"], got[name + "_scale"] = codes, scale
    return got


def _exact_attention(st, case):
    block, nq = case["block"], case["queries"]
    H, G, D = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"]
    lens, tables = st["lens"].cpu().tolist(), st["tables"].long()
    out = torch.zeros(case["sequences"] * nq, H * G, D, dtype=torch.float64, device=DEV)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for r, n in enumerate(lens):
        t = tables[r, :-(-n // block)]
        k, v = (((st[x + "_cache"].view(torch.uint8)[t].view(CODES[case["format"]]).double()
                  * st[x + "_scale"][t].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n])
                for x in ("k", "v"))
        for i in range(nq):
            sees = n - nq + i + 1
            if sees < 1:
                continue
            q = st["q"][r * nq + i].double().view(H, G, D)
            s = torch.einsum("hgd,hnd->hgn", q, k[:, :sees]) * st["scale"]
            lse[r * nq + i] = torch.logsumexp(s, -1).reshape(-1)
            out[r * nq + i] = torch.einsum("hgn,hnd->hgd", torch.softmax(s, -1), v[:, :sees]).reshape(H * G, D)
    return {"out": out, "lse": lse}
