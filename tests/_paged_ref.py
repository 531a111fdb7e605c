"""Plain 64-bit restatements of the paged 8-bit cache's operators, for the tests."""

import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def round_code(x, fmt):
    """float64 values to the nearest value of the format, ties to even."""
    if fmt == torch.int8:
        return x.round()
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return (x / step).round() * step


def block_scale(amax, fmt):
    """Smallest power of two >= 2^-126 with amax / scale <= the format's largest value; NaN if not finite."""
    if not math.isfinite(amax):
        return math.nan
    m, e = math.frexp(amax)              # amax = m 2^e
    lm, le = math.frexp(LARGEST[fmt])
    return math.ldexp(1.0, max(-126, e - le + (1 if m > lm else 0)) if amax > 0 else -126)


class RefCache:
    """One layer's values as a dictionary block -> per head (scale, {place: codes})."""

    def __init__(self, heads, block, fmt):
        self.heads, self.block, self.fmt = heads, block, fmt
        self.scale, self.codes = {}, {}

    def write(self, x, slots):
        """x [T, heads, D] float64 on the CPU, slots a list; runs of neighbours in one block."""
        t = 0
        while t < len(slots):
            if slots[t] < 0:
                t += 1
                continue
            b, z = slots[t] // self.block, t
            while z < len(slots) and slots[z] >= 0 and slots[z] // self.block == b:
                z += 1
            places = [s % self.block for s in slots[t:z]]
            anew = 0 in places
            for h in range(self.heads):
                rows = x[t:z, h]
                amax = float(rows.abs().max()) if torch.isfinite(rows).all() else math.inf
                scale = block_scale(amax, self.fmt)
                old = None if anew else self.scale.get((b, h))
                if old is not None:
                    scale = math.nan if math.isnan(old) or math.isnan(scale) else max(old, scale)
                held = {} if anew else dict(self.codes.get((b, h), {}))
                if old is not None and scale > old:
                    held = {p: round_code(c * (old / scale), self.fmt) for p, c in held.items()}
                for i, p in enumerate(places):
                    held[p] = torch.zeros_like(rows[i]) if math.isnan(scale) else round_code(rows[i] / scale, self.fmt)
                self.scale[b, h], self.codes[b, h] = scale, held
            t = z

    def read(self, slots, dim):
        out = torch.zeros(len(slots), self.heads, dim, dtype=torch.float64)
        for t, s in enumerate(slots):
            if s >= 0:
                b, p = s // self.block, s % self.block
                for h in range(self.heads):
                    out[t, h] = self.codes[b, h][p] * self.scale[b, h]
        return out


class RefTables:
    """Block tables with a free stack, in Python."""

    def __init__(self, lens, tables, free, block):
        self.lens, self.tables, self.free, self.block = list(lens), [list(t) for t in tables], list(free), block

    def step(self, new, total, shift):
        b, R = self.block, len(self.lens)
        for r in range(R):
            if new[r] < 0:
                self.free += self.tables[r][:-(-self.lens[r] // b)]
        cu, slots, positions, granted, short = [0], [], [], [], False
        lens = list(self.lens)
        for r in range(R):
            n = max(new[r], 0)
            cu.append(cu[-1] + n)
            have, want = -(-self.lens[r] // b), -(-(self.lens[r] + n) // b)
            ok = new[r] >= 0 and want <= len(self.tables[r])
            if ok and want > have:
                short = short or want - have > len(self.free)
                ok = not short
                if ok:
                    for c in range(have, want):
                        self.tables[r][c] = self.free.pop()
            granted.append(n if ok else 0)
            lens[r] = 0 if new[r] < 0 else self.lens[r] + granted[r]
            for i in range(n):
                p = self.lens[r] + i
                slots.append(self.tables[r][p // b] * b + p % b if ok else -1)
                positions.append(p + shift[r])
        self.lens = lens
        pad = max(0, total - len(slots))
        return dict(lens=lens, cu=cu, slots=(slots + [-1] * pad)[:total], positions=(positions + [0] * pad)[:total],
                    granted=granted)


def rotary(x, positions, inv_freq, interleaved, factor, inverse):
    """x [T, H, D] float64; complex multiplication of the pairs."""
    d = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq
    turn = torch.polar(torch.full_like(angle, factor), -angle if inverse else angle)[:, None]
    y = x.double().clone()
    head = y[..., :d]
    pairs = head.unflatten(-1, (d // 2, 2)) if interleaved else head.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y[..., :d] = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return y


def attention(q, k, v, scale, causal):
    """One sequence: q [m, H, D], k / v [n, Hkv, D], float64.  (out [m, H, D], lse [m, H])."""
    m, H, D = q.shape
    n, Hk = k.shape[:2]
    out = torch.zeros(m, H, D, dtype=torch.float64, device=q.device)
    lse = torch.full((m, H), -math.inf, dtype=torch.float64, device=q.device)
    for i in range(m):
        sees = n - m + i + 1 if causal else n
        if sees < 1:
            continue
        kk, vv = (x[:sees].repeat_interleave(H // Hk, 1) for x in (k, v))
        s = torch.einsum("hd,nhd->hn", q[i], kk) * scale
        lse[i] = torch.logsumexp(s, -1)
        out[i] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vv)
    return out, lse
