"""Plain 64-bit restatement of the 8-bit KV cache operators and of the q / k norm with rotation, for the tests."""
import math

import torch

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}     # a rounding's error relative to the value


def e4m3(x):
    """Nearest e4m3 value, ties to even (|x| at most 464; NaN stays NaN)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exponent_of(amax):
    """Least e >= -126 with amax <= 448 * 2^e."""
    if amax == 0:
        return -126
    m, x = math.frexp(amax)                 # m in [0.5, 1)
    return max(-126, x - 9 + (1 if m > 0.875 else 0))


class Cache:
    """A cache on the GPU with its host mirror in 64 bits: codes' values and scales' exponents."""

    def __init__(self, b, cap, hk, d, blk, page=0, extra_pages=2, seed=0, filled=False, batch_rows=None):
        g = torch.Generator().manual_seed(seed)
        self.b, self.hk, self.d, self.blk, self.page = b, hk, d, blk, page
        if page:
            self.rows, self.per = page, -(-cap // page)
            n = b * self.per + extra_pages
            self.table = torch.randperm(n, generator=g)[:b * self.per].view(b, self.per).to(torch.int32)
        else:
            self.rows, self.per = -(-cap // blk) * blk, 1
            n = b if batch_rows is None else batch_rows
            self.table = None
        self.cap = self.rows * self.per
        # codes: any finite byte; scales: exponents around 0
        self.codes = [torch.randint(0, 256, (n, self.rows, hk, d), generator=g, dtype=torch.int32) for _ in range(2)]
        for c in self.codes:
            c[(c & 127) == 127] = 0x31
        self.scales = [torch.randint(120, 124, (n, self.rows // blk, hk), generator=g, dtype=torch.int32) for _ in range(2)]

    def gpu(self):
        """k_cache, v_cache, k_scale, v_scale"""
        c = [x.to(torch.uint8).cuda().view(torch.float8_e4m3fn) for x in self.codes]
        s = [x.to(torch.uint8).cuda().view(torch.float8_e8m0fnu) for x in self.scales]
        return c[0], c[1], s[0], s[1]

    def block_table(self):
        return None if self.table is None else self.table.cuda()

    def place(self, i, tok, rows_of=None):
        if self.table is None:
            return (i if rows_of is None else int(rows_of[i])), tok
        return int(self.table[i, tok // self.page]), tok % self.page

    def values(self, which, i, n, rows_of=None):
        """(n, hk, d) in 64 bits: what the first n tokens of sequence i stand for."""
        if self.table is None:
            idx = torch.tensor([i if rows_of is None else int(rows_of[i])])
        else:
            idx = self.table[i, :-(-n // self.page)].long()
        v = decode(self.codes[which][idx]).flatten(0, 1)
        s = torch.exp2(self.scales[which][idx].double() - 127).repeat_interleave(self.blk, 1).flatten(0, 1)
        return (v * s[..., None])[:n]


def decode(c):
    """e4m3 codes (whole numbers) -> 64-bit values"""
    return c.to(torch.uint8).view(torch.float8_e4m3fn).double()


def encode(v):
    """e4m3 values in 64 bits -> codes"""
    return v.float().to(torch.float8_e4m3fn).view(torch.uint8).to(torch.int32)


def write_ref(cache, which, i, start, x, dtype, rows_of=None):
    """Sequence i's new tokens x (n, hk, d) at start, by the definition, into the host mirror."""
    x = x.double()
    top = 120 if dtype == "bf16" else 8
    end = min(start + x.shape[0], cache.cap)
    at = start
    while at < end:
        lo = at // cache.blk * cache.blk
        hi = min(end, lo + cache.blk)
        page, row = cache.place(i, lo, rows_of)
        new = x[at - start:hi - start]
        for h in range(cache.hk):
            y = new[:, h]
            fin = y[torch.isfinite(y)]
            e = exponent_of(float(fin.abs().max()) if fin.numel() else 0.0)
            was = int(cache.scales[which][page, row // cache.blk, h]) - 127
            if at > lo:
                e = max(e, was)
                if e > was:
                    held = cache.codes[which][page, row:row + at - lo, h]
                    nan = (held & 127) == 127
                    again = encode(e4m3(decode(held).nan_to_num(0.0) * 2.0 ** (was - e)))
                    sign = held & 128       # (a value that rounds to zero keeps its sign)
                    cache.codes[which][page, row:row + at - lo, h] = torch.where(nan, held, again & 127 | sign)
            z = y * 2.0 ** -e
            lim = 240.0 if e >= top else 448.0
            c = encode(e4m3(z.nan_to_num(0.0, 0.0, 0.0)).clamp(-lim, lim)) & 127
            sign = torch.signbit(y).to(torch.int32) << 7
            c = torch.where(torch.isfinite(y), c | sign, 127 | sign)
            cache.codes[which][page, row + at - lo:row + hi - lo, h] = c
            cache.scales[which][page, row // cache.blk, h] = e + 127
        at = hi


def attend_ref(q, k, v, causal=False, window=(-1, -1), slopes=None, scale=None, dtype="bf16"):
    """One sequence: q (m, h, d), k / v (n, hk, d), 64 bits.  Returns out (m, h, d) and, element by element, how far a
    kernel may be off that rounds P and the result once to 16 bits and forms the scores in fp32.

    With half step u: the result's rounding gives u |o|; rounding p_j gives u p_j |v_j| each; a score off by ds makes
    p_j off by a factor of ds and the sum of p by as much, 2 ds in all, where ds <= scale d 2^-24 sum |q||k| (fp32 sum of
    d exact products) plus 2^-20 for the exponential, the mask's bias and the sums of P; in fp16 a P under 2^-14 is
    off by up to 2^-25 of the row's largest."""
    u = HALF_STEP[dtype]
    (m, h, d), (n, hk) = q.shape, k.shape[:2]
    scale = d ** -0.5 if scale is None else scale
    q = q.double()
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    i, j = torch.arange(m)[:, None] + n - m, torch.arange(n)[None, :]
    i, j = i.to(q.device), j.to(q.device)
    hide = torch.zeros(m, n, dtype=torch.bool, device=q.device)
    if causal:
        window = (window[0], 0)
    if window[1] >= 0:
        hide |= j > i + window[1]
    if window[0] >= 0:
        hide |= j < i - window[0]
    outs, tols = [], []
    for a in range(h):
        kk, vv = k[:, a // (h // hk)].to(q.device).double(), v[:, a // (h // hk)].to(q.device).double()
        # (values no row sees do not matter, whatever they are)
        seen = (~hide).any(0)
        kk, vv = torch.where(seen[:, None], kk, 0.0), torch.where(seen[:, None], vv, 0.0)
        s = (q[:, a] @ kk.t().contiguous()) * scale
        ds = (q[:, a].abs() @ kk.t().abs().contiguous()) * scale * d * 2.0 ** -24
        if slopes is not None:
            s = s - float(slopes[a]) * (i - j).abs()
            ds = ds + abs(float(slopes[a])) * n * 2.0 ** -22
        ds = ds.masked_fill(hide, 0.0).amax(1, keepdim=True) + 2.0 ** -20
        s = s.masked_fill(hide, -math.inf)
        top = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
        l = p.sum(1, keepdim=True)
        p = torch.where(l > 0, p / l, 0.0)
        o = p @ vv
        reach = p @ vv.abs()
        tol = u * o.abs() + (u + 2 * ds) * (1 + 4 * u) * reach
        if dtype == "fp16":
            tol = tol + (~hide).double() @ vv.abs() * 2.0 ** -25 / l.clamp_min(1.0) + 2.0 ** -25
        outs.append(o)
        tols.append(tol)
    return torch.stack(outs, 1), torch.stack(tols, 1)


def norm_rotary_ref(x, w, cos, sin, pos, eps, inter):
    """x (b, s, h, d) 64 bits; cos / sin (b, s, rd / 2) rows of the tokens' positions; differentiable."""
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    rd = 2 * cos.shape[-1]
    c, s = cos[:, :, None], sin[:, :, None]
    if inter:
        a, b = n[..., 0:rd:2], n[..., 1:rd:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = n[..., :rd // 2], n[..., rd // 2:rd]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, n[..., rd:]), -1)
