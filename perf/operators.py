"""Measured cases of the operators around an 8-bit KV cache: the norm and rotation of query and key heads in
one pass (with its backward), writing tokens to a cache of e4m3 codes with one power-of-two scale per block of
tokens and head, reading such a cache back, and attention over it.

`own` selects the framework's operators; without it every operator is computed in its plain form, elementary
torch operations in 32 bits."""
import math
import os
import sys

import torch

own = False
_package = None

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
LEAST_EXPONENT = -126   # of a block's scale; an all-zero block has it too


# ------------------------------------------------------------------------------------------- cases
def listed():
    norm = dict(op="norm", inter=False, table="fp32")
    attend = dict(op="attend", ragged=False, append=False, causal=True, window=-1)
    return [
        # one decode step of a batch: q and k slices of a packed projection, positions from the cache's lengths
        dict(norm, name="norm decode 64", b=64, s=1, h=32, hk=8, d=128, rd=128, dtype="bf16", train=False),
        # a training step's q and k, forward and backward
        dict(norm, name="norm train 4096", b=4, s=4096, h=32, hk=8, d=128, rd=128, dtype="bf16", train=True),
        # odd token count, partial rotation of interleaved pairs, a table in the tensors' type
        dict(norm, name="norm train odd", b=1, s=2731, h=12, hk=12, d=96, rd=64, dtype="fp16", train=True, inter=True, table="same"),
        # one token of every sequence of a decode batch into a paged cache
        dict(op="write", name="write decode 128", b=128, new=1, new_lo=1, kv=2048, kv_lo=200, hk=8, d=128, page=16, block=16, dtype="fp16"),
        # prompts of uneven length into pages of 64 with a scale every 32 tokens
        dict(op="write", name="write prompts", b=8, new=4000, new_lo=37, kv=4096, kv_lo=0, hk=8, d=128, page=64, block=32, dtype="bf16"),
        # a small cache back into 16 bits (the cached prefix of a short chunk)
        dict(op="read", name="read short", b=4, kv=777, kv_lo=1, hk=4, d=64, page=16, block=16, dtype="fp16", ragged=False),
        # long cached prefixes into one ragged tensor
        dict(op="read", name="read ragged", b=32, kv=8192, kv_lo=500, hk=8, d=128, page=64, block=64, dtype="bf16", ragged=True),
        # one long sequence, one token: the keys have to be split over the chip
        dict(attend, name="attend one long", b=1, sq=1, kv=65536, kv_lo=65536, h=32, hk=8, d=128, page=64, block=64, dtype="bf16"),
        # the framework's decode benchmark with an 8-bit cache
        dict(attend, name="attend decode 128", b=128, sq=1, kv=8192, kv_lo=8192, h=32, hk=8, d=128, page=0, block=64, dtype="fp16"),
        # a serving step: the new token is written, then attended, over lengths that differ
        dict(attend, name="attend append", b=48, sq=1, kv=4096, kv_lo=100, h=16, hk=16, d=64, page=16, block=16, dtype="bf16", append=True),
        # drafted tokens against a sliding window, wide heads
        dict(attend, name="attend drafted", b=24, sq=5, kv=6000, kv_lo=900, h=8, hk=2, d=256, page=32, block=32, dtype="bf16", window=4095),
        # chunks of prompts and single tokens in one ragged batch
        dict(attend, name="attend ragged", b=16, sq=1024, kv=8192, kv_lo=1200, h=32, hk=8, d=128, page=64, block=64, dtype="bf16", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "write", "read", "attend", "attend"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        d = rng.choice([64, 80, 96, 128, 192, 256])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([1, 2, 4, 8])
        most = 4 * 4096 * 40 * 128 // ((h + hk) * d)
        b = _log_int(rng, 1, 64)
        s = _log_int(rng, 1, max(1, min(8192, most // b)))
        rd = rng.choice([d, d // 2 // 16 * 16])
        return dict(op=op, b=b, s=s, h=h, hk=hk, d=d, rd=rd, dtype=dtype, train=rng.random() < 0.6,
                    inter=rng.random() < 0.5, table=rng.choice(["fp32", "same"]))
    d = rng.choice([64, 80, 96, 128, 192, 256])
    hk = rng.choice([1, 2, 4, 8, 16])
    block = rng.choice([16, 32, 64, 128])
    page = rng.choice([0, block, block * rng.choice([2, 3, 4])])
    if op == "attend":
        group = rng.choice([1, 2, 4, 7, 8])
        b = _log_int(rng, 1, 128)
        ragged = rng.random() < 0.3
        kv = _log_int(rng, 64, min(32768, (64 * 8192 * 8 * 128) // (b * hk * d) + 64))
        sq = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 2, min(kv, 1024))])
        # (the plain form holds every score: rows x keys of all heads)
        sq = max(1, min(sq, kv, (1 << 29) // (b * hk * group * kv)))
        kv_lo = rng.randint(sq, kv)
        return dict(op=op, b=b, sq=sq, kv=kv, kv_lo=kv_lo, h=hk * group, hk=hk, d=d, page=page, block=block,
                    dtype=dtype, ragged=ragged, append=not ragged and rng.random() < 0.3,
                    causal=rng.random() < 0.7, window=rng.choice([-1, -1, rng.randint(0, kv)]))
    b = _log_int(rng, 1, 64)
    kv = _log_int(rng, 64, min(16384, (32 * 8192 * 8 * 128) // (b * hk * d) + 64))
    if op == "read":
        return dict(op=op, b=b, kv=kv, kv_lo=rng.randint(0, kv), hk=hk, d=d, page=page, block=block, dtype=dtype,
                    ragged=rng.random() < 0.5)
    kv = min(kv, 2048)
    new = rng.choice([1, rng.randint(1, 16), _log_int(rng, 1, kv)])
    return dict(op=op, b=b, new=new, new_lo=rng.randint(0, new), kv=kv, kv_lo=rng.randint(0, kv - new), hk=hk, d=d,
                page=page, block=block, dtype=dtype)


# ------------------------------------------------------------------------------------------- inputs
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread: what a case costs does not hang on the seed."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _shuffled(values, gen):
    return [values[i] for i in torch.randperm(len(values), generator=gen).tolist()]


def _exponent(amax):
    """Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), not under LEAST_EXPONENT."""
    m, x = torch.frexp(amax)              # amax = m 2^x, m in [0.5, 1)
    e = x - 9 + (m > 0.875)
    return torch.where(amax > 0, e, LEAST_EXPONENT).clamp_min(LEAST_EXPONENT)


def _pow2(e):
    """2^e, by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _rows_of(case):
    """(rows of a page, pages of a sequence): a contiguous cache is one page per sequence."""
    if case["page"]:
        return case["page"], -(-case["kv"] // case["page"])
    return -(-case["kv"] // case["block"]) * case["block"], 1


def _lengths(case):
    """Cached tokens before the call, per sequence."""
    lo, hi = case["kv_lo"], case["kv"]
    if case["op"] == "write":
        return _spread(lo, hi - case["new"], case["b"])
    if case["op"] == "attend" and case["append"]:
        return _spread(lo - case["sq"], hi - case["sq"], case["b"])
    return _spread(lo, hi, case["b"])


def _news(case):
    """New tokens (write) or query tokens (attend) per sequence."""
    if case["op"] == "write":
        return _spread(case["new_lo"], case["new"], case["b"])
    if case.get("ragged"):   # mostly single tokens, every fourth sequence a chunk
        return [case["sq"] - case["sq"] * (i // 4) // case["b"] if i % 4 == 0 else 1 for i in range(case["b"])]
    return [case["sq"]] * case["b"]


def _make_cache(case, g):
    """Codes and scales of a filled cache: channels of different size, some loud tokens."""
    rows, per = _rows_of(case)
    pages = case["b"] * per + (3 if case["page"] else 0)
    block, hk, d = case["block"], case["hk"], case["d"]
    made = []
    for _ in range(2):
        size = torch.exp(0.7 * torch.randn(hk, d, device="cuda", generator=g))
        loud = 1 + 6 * (torch.rand(pages, rows, hk, 1, device="cuda", generator=g) > 0.97).float()
        x = torch.randn(pages, rows, hk, d, device="cuda", generator=g).mul_(size).mul_(loud)
        x = x.view(pages, rows // block, block, hk, d)
        e = _exponent(x.abs().amax((2, 4)))
        codes = x.mul_(_pow2(-e)[:, :, None, :, None]).view(pages, rows, hk, d).to(torch.float8_e4m3fn)
        made.append((codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)))
    return made


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    hg = torch.Generator().manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["op"] == "norm":
        b, s, h, hk, d, rd = (case[n] for n in ("b", "s", "h", "hk", "d", "rd"))
        qkv = torch.randn(b, s, (h + 2 * hk) * d, device="cuda", generator=g).mul_(1.7).to(dt)
        q = qkv[..., :h * d].view(b, s, h, d).detach().requires_grad_(case["train"])
        k = qkv[..., h * d:(h + hk) * d].view(b, s, hk, d).detach().requires_grad_(case["train"])
        w = [(1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dt).requires_grad_(case["train"]) for _ in range(2)]
        table = 8192 if s == 1 else s
        angle = torch.arange(table, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / max(rd, 1))
        tdt = torch.float32 if case["table"] == "fp32" else dt
        st.update(q=q, k=k, w=w, cos=angle.cos().to("cuda", tdt), sin=angle.sin().to("cuda", tdt), positions=None)
        if s == 1:   # a decode step: every row at its sequence's own position
            st["positions"] = torch.randint(0, table, (b, s), device="cuda", generator=g, dtype=torch.int32)
        if case["train"]:
            st["grads"] = [torch.randn(b, s, n, d, device="cuda", generator=g).to(dt) for n in (h, hk)]
        return st
    (st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"]) = _make_cache(case, g)
    st["order"] = order = _shuffled(list(range(case["b"])), hg)
    lens = [_lengths(case)[i] for i in order]
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["table"] = None
    if case["page"]:
        per = _rows_of(case)[1]
        ids = torch.randperm(case["b"] * per + 3, generator=hg)[:case["b"] * per]
        st["table"] = ids.view(case["b"], per).to(torch.int32).cuda()
    hk, d = case["hk"], case["d"]
    if case["op"] == "read":
        if case["ragged"]:
            st["cu"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
            st["total"] = sum(lens)
        return st
    news = [_news(case)[i] for i in order]
    st["news"], most = news, max(news)
    st["cu"] = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
    size = torch.exp(0.7 * torch.randn(hk, d, device="cuda", generator=g))
    if case["op"] == "write":
        st["kv"] = [torch.randn(sum(news), hk, d, device="cuda", generator=g).mul(size).to(dt) for _ in range(2)]
        st["most"] = most
        return st
    shape = (sum(news), case["h"], d) if case["ragged"] else (case["b"], case["sq"], case["h"], d)
    st["q"] = torch.randn(shape, device="cuda", generator=g).to(dt)
    if case["append"]:
        st["kv"] = [torch.randn(case["b"], case["sq"], hk, d, device="cuda", generator=g).mul(size).to(dt) for _ in range(2)]
    return st


# ------------------------------------------------------------------------------------------- the operators
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _framework():
    global _package
    if _package is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-flash-attention_amd"))
        import vllm_flash_attn as _package
    return _package


def _run_own(st):
    fa, case = _framework(), st["case"]
    if case["op"] == "norm":
        out = fa.qk_norm_rotary_func(st["q"], st["k"], st["w"][0], st["w"][1], st["cos"], st["sin"], positions=st["positions"],
                                     eps=1e-6, rotary_interleaved=case["inter"])
        if not case["train"]:
            return out
        return (*(o.detach() for o in out), *torch.autograd.grad(out, (st["q"], st["k"], *st["w"]), st["grads"]))
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if case["op"] == "write":
        fa.quantize_kvcache(*st["kv"], *cache, st["lens"], block_table=st["table"], cu_seqlens=st["cu"], max_seqlen=st["most"])
        return cache
    if case["op"] == "read":
        if case["ragged"]:
            return fa.dequantize_kvcache(*cache, st["lens"], cu_seqlens=st["cu"], total_seqlen=st["total"], block_table=st["table"],
                                         dtype=DTYPES[case["dtype"]])
        return fa.dequantize_kvcache(*cache, st["lens"], max_seqlen=case["kv"], block_table=st["table"], dtype=DTYPES[case["dtype"]])
    kw = dict(cache_seqlens=st["lens"], block_table=st["table"], causal=case["causal"], window_size=(case["window"], -1))
    if case["ragged"]:
        kw.update(cu_seqlens_q=st["cu"], max_seqlen_q=max(st["news"]))
    if case["append"]:
        kw.update(k=st["kv"][0], v=st["kv"][1])
    out = fa.flash_attn_with_quantized_kvcache(st["q"], *cache, **kw)
    return (out, *cache) if case["append"] else out


def _run_plain(st):
    case = st["case"]
    if case["op"] == "norm":
        q, k, (wq, wk) = st["q"], st["k"], st["w"]
        cos, sin = st["cos"].float(), st["sin"].float()
        if st["positions"] is None:
            cos, sin = cos[None, :, None, :], sin[None, :, None, :]
        else:
            at = st["positions"].long()
            cos, sin = cos[at][:, :, None, :], sin[at][:, :, None, :]
        out = (_norm_rotary(q, wq, cos, sin, case["inter"]), _norm_rotary(k, wk, cos, sin, case["inter"]))
        if not case["train"]:
            return out
        return (*(o.detach() for o in out), *torch.autograd.grad(out, (q, k, wq, wk), st["grads"]))
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if case["op"] == "write":
        _write(st, st["kv"][0], st["k_cache"], st["k_scale"])
        _write(st, st["kv"][1], st["v_cache"], st["v_scale"])
        return cache
    if case["op"] == "read":
        dt = DTYPES[case["dtype"]]
        made = [_read(st, c, s, st["lens"], case["kv"]) for c, s in (cache[0::2], cache[1::2])]
        if case["ragged"]:
            at = torch.arange(st["total"], device="cuda")
            seq = torch.searchsorted(st["cu"][1:].long(), at, right=True)
            return tuple(x[seq, at - st["cu"].long()[seq]].to(dt) for x in made)
        return tuple(x.to(dt) for x in made)
    lens = st["lens"]
    if case["append"]:
        _write(st, st["kv"][0].flatten(0, 1), st["k_cache"], st["k_scale"])
        _write(st, st["kv"][1].flatten(0, 1), st["v_cache"], st["v_scale"])
        lens = lens + case["sq"]
    out = _attend(st, lens)
    return (out, *cache) if case["append"] else out


def _norm_rotary(x, w, cos, sin, inter):
    dt, x = x.dtype, x.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
    rd = 2 * cos.shape[-1]
    a, b = (n[..., 0:rd:2], n[..., 1:rd:2]) if inter else (n[..., :rd // 2], n[..., rd // 2:rd])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if inter else torch.cat(y, -1)
    return torch.cat((y, n[..., rd:]), -1).to(dt)


def _flat_rows(st, pos):
    """Rows of the flattened cache that hold the positions pos (b, n)."""
    rows, _ = _rows_of(st["case"])
    if st["table"] is None:
        return torch.arange(pos.shape[0], device="cuda")[:, None] * rows + pos
    return st["table"].long().gather(1, pos // rows) * rows + pos % rows


def _write(st, x, cache, scale):
    case = st["case"]
    block, (b, hk, d) = case["block"], (case["b"], case["hk"], case["d"])
    start, cu = st["lens"].long(), st["cu"].long()
    new = cu[1:] - cu[:-1]
    most = (max(st["news"]) + block - 2) // block + 1
    first = start // block
    last = torch.maximum(start + new - 1, torch.zeros_like(start)) // block
    blk = torch.minimum(first[:, None] + torch.arange(most, device="cuda"), last[:, None])   # (a block written twice gets the same twice)
    pos = (blk[:, :, None] * block + torch.arange(block, device="cuda")).view(b, -1)
    old = pos < start[:, None]
    fresh = ~old & (pos < (start + new)[:, None])
    src = (cu[:-1, None] + pos - start[:, None]).clamp(0, max(0, x.shape[0] - 1))
    at = _flat_rows(st, pos)
    codes, scales = cache.view(torch.uint8).view(-1, hk, d), scale.view(torch.uint8).view(-1, hk)
    were = codes[at]
    value = torch.where(fresh[..., None, None], x[src].float() if x.shape[0] else torch.zeros((), device="cuda"), 0.0)
    e_new = _exponent(value.view(b, most, block, hk, d).abs().amax((2, 4)))
    at_block = at.view(b, most, block)[:, :, 0] // block
    e_old = scales[at_block].int() - 127
    holds = (blk * block < start[:, None])[..., None]
    e = torch.where(holds, torch.maximum(e_old, e_new), e_new)
    e = torch.where((new > 0)[:, None, None], e, e_old)

    def rows(t):
        return t[:, :, None, :].expand(b, most, block, hk).reshape(b, -1, hk, 1)

    kept = were.view(torch.float8_e4m3fn).float() * rows(_pow2(e_old - e))
    y = torch.where(fresh[..., None, None], value * rows(_pow2(-e)), kept).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[at] = torch.where((fresh | old)[..., None, None], y, were)
    scales[at_block] = (e + 127).to(torch.uint8)


def _read(st, cache, scale, lens, most):
    """(b, most, hk, d) in 32 bits, zeros behind each sequence."""
    case = st["case"]
    pos = torch.arange(most, device="cuda").expand(case["b"], most)
    at = _flat_rows(st, pos)
    hk, d = case["hk"], case["d"]
    x = cache.view(torch.uint8).view(-1, hk, d)[at].view(torch.float8_e4m3fn).float()
    x = x * scale.view(torch.uint8).view(-1, hk)[at // case["block"]].view(torch.float8_e8m0fnu).float()[..., None]
    return torch.where((pos < lens[:, None])[..., None, None], x, 0.0)


def _attend(st, lens):
    case = st["case"]
    b, h, hk, d, kv = (case[n] for n in ("b", "h", "hk", "d", "kv"))
    k = _read(st, st["k_cache"], st["k_scale"], lens, kv)
    v = _read(st, st["v_cache"], st["v_scale"], lens, kv)
    sq, q = max(st["news"]), st["q"].float()
    nq = (st["cu"][1:] - st["cu"][:-1]).long()
    if case["ragged"]:
        i = torch.arange(sq, device="cuda")
        src = (st["cu"][:-1].long()[:, None] + i).clamp_max(q.shape[0] - 1)
        q = torch.where((i < nq[:, None])[..., None, None], q[src], 0.0)
    q = q.view(b, sq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    s = q @ k.permute(0, 2, 3, 1).contiguous() * d ** -0.5
    i, j = torch.arange(sq, device="cuda")[:, None], torch.arange(kv, device="cuda")
    shift = (lens.long() - nq)[:, None, None]
    seen = (j < lens[:, None, None]).expand(b, sq, kv)
    if case["causal"]:
        seen = seen & (j <= i + shift)
    if case["window"] >= 0:
        seen = seen & (j >= i + shift - case["window"])
    s = s.view(b, hk, -1, sq, kv).masked_fill_(~seen[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    total = s.sum(-1, keepdim=True)
    o = s.view(b, hk, -1, kv) @ v.permute(0, 2, 1, 3).contiguous()
    o = (o / total.clamp_min(1e-30).view(b, hk, -1, 1)).view(b, hk, -1, sq, d).permute(0, 3, 1, 2, 4).reshape(b, sq, h, d).to(st["q"].dtype)
    if not case["ragged"]:
        return o
    at = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(st["cu"][1:].long(), at, right=True)
    return o[seq, at - st["cu"].long()[seq]]


# ------------------------------------------------------------------------------------------- what a pass costs
def work(case):
    if case["op"] == "norm":
        n = case["b"] * case["s"] * (case["h"] + case["hk"]) * case["d"]
        table = (case["b"] if case["s"] == 1 else case["s"]) * case["rd"] * (4 if case["table"] == "fp32" else 2)
        return {"bytes": n * (8 if case["train"] else 4) + table, "flops": n * (30 if case["train"] else 10)}
    lens, hk, d = _lengths(case), case["hk"], case["d"]
    if case["op"] == "write":
        n = sum(_news(case)) * hk * d
        return {"bytes": 2 * n * 3, "flops": 2 * n * 3}
    if case["op"] == "read":
        n = sum(lens) * hk * d
        rows = sum(lens) if case["ragged"] else case["b"] * case["kv"]
        return {"bytes": 2 * n + 4 * rows * hk * d, "flops": 2 * n}
    news = _news(case)
    if case["append"]:
        lens = [n + case["sq"] for n in lens]
    keys = pairs = 0
    for n, m in zip(lens, news):
        lo = 0 if case["window"] < 0 else max(0, n - m - case["window"])
        keys += n - lo
        first = n - m + 1 if case["causal"] else n        # keys that the first query row sees, without a window
        for i in range(m):
            hi = first + i if case["causal"] else n
            pairs += hi - (0 if case["window"] < 0 else max(0, n - m + i - case["window"]))
    rows = sum(news) * case["h"]
    extra = 2 * sum(news) * hk * d * 3 if case["append"] else 0
    return {"bytes": 2 * keys * hk * d + 2 * keys // case["block"] * hk + 4 * rows * d + extra, "flops": 4 * pairs * case["h"] * d}


# ------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(st)
    if case["op"] == "write":
        return _exact_write(st)
    if case["op"] == "read":
        k, v = (_exact_sequences(st, n, [int(x) for x in st["lens"]]) for n in "kv")
        if case["ragged"]:
            return torch.cat(k), torch.cat(v)
        pad = [torch.zeros(case["b"], case["kv"], case["hk"], case["d"], dtype=torch.float64, device="cuda") for _ in range(2)]
        for p, seqs in zip(pad, (k, v)):
            for i, x in enumerate(seqs):
                p[i, :x.shape[0]] = x
        return tuple(pad)
    lens = [int(x) for x in st["lens"]]
    if sum(lens) * case["hk"] * case["d"] * 16 > 64e9 or case["b"] * case["hk"] > 2048:
        return None
    cache = ()
    if case["append"]:
        cache = _exact_write(st, apply=True)
        lens = [n + case["sq"] for n in lens]
    return (_exact_attend(st, lens), *cache) if case["append"] else _exact_attend(st, lens)


def _exact_norm(st):
    """The formulas with the rotation as complex numbers; gradients in closed form."""
    case, out, grads = st["case"], [], []
    turn = torch.complex(st["cos"].double(), st["sin"].double())
    turn = turn[None] if st["positions"] is None else turn[st["positions"].long()]
    rd, half = case["rd"], case["rd"] // 2

    def rotate(x, by):
        if case["inter"]:
            z = torch.view_as_complex(x[..., :rd].unflatten(-1, (half, 2)).contiguous()) * by[:, :, None]
            return torch.cat((torch.view_as_real(z).flatten(-2), x[..., rd:]), -1)
        z = torch.complex(x[..., :half].contiguous(), x[..., half:rd].contiguous()) * by[:, :, None]
        return torch.cat((z.real, z.imag, x[..., rd:]), -1)

    for i, n in enumerate("qk"):
        x, w = st[n].detach().double(), st["w"][i].detach().double()
        r = 1 / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        out.append(rotate(x * r * w, turn))
        if case["train"]:
            g = rotate(st["grads"][i].double(), turn.conj())
            grads.append((r * (g * w - x * r * (g * w * x * r).mean(-1, keepdim=True)), (g * x * r).sum((0, 1, 2))))
    if not case["train"]:
        return tuple(out)
    return (*out, grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _e4m3_values(x):
    """x rounded to the nearest e4m3 value, ties to even: three bits behind the leading one, steps of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _place(st, i, j):
    """(page, row in it) of position j of sequence i."""
    rows, _ = _rows_of(st["case"])
    return (i, j) if st["table"] is None else (int(st["table_host"][i][j // rows]), j % rows)


def _exact_write(st, apply=False):
    case = st["case"]
    st["table_host"] = None if st["table"] is None else st["table"].tolist()
    lens, block, cu = [int(x) for x in st["lens"]], case["block"], st["cu"].tolist()
    out = []
    for x, name in zip(st["kv"], "kv"):
        x = x.reshape(-1, case["hk"], case["d"]).double()
        values = st[name + "_cache"].double()
        scales = st[name + "_scale"].double()
        for i, n in enumerate(lens):
            m = cu[i + 1] - cu[i]
            at = n
            while at < n + m:
                low = at // block * block
                high = min(low + block, n + m)
                new = x[cu[i] + at - n:cu[i] + high - n]
                page, row = _place(st, i, low)
                top = new.abs().amax((0, 2))
                e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -140) / E4M3_MAX)).clamp_min(LEAST_EXPONENT)
                s, was = torch.exp2(e), scales[page, row // block].clone()
                if at > low:
                    s = torch.maximum(s, was)
                    held = values[page, row:row + at - low]
                    values[page, row:row + at - low] = _e4m3_values(held * (was / s)[:, None])
                scales[page, row // block] = s
                values[page, row + at - low:row + high - low] = _e4m3_values(new / s[:, None])
                at = high
        out.append((values, scales))
    if apply:
        for (values, scales), name in zip(out, "kv"):
            st[name + "_exact"] = (values, scales)
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_sequences(st, name, lens):
    """The values of every sequence, (length, hk, d) each."""
    case, (rows, _) = st["case"], _rows_of(st["case"])
    values, scales = st.get(name + "_exact") or (st[name + "_cache"], st[name + "_scale"])
    seqs = []
    for i, n in enumerate(lens):
        pages = [i] if st["table"] is None else st["table"][i, :-(-n // rows)].long()
        x = values[pages] if values.dtype == torch.float64 else values.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
        s = scales[pages] if scales.dtype == torch.float64 else scales.view(torch.uint8)[pages].view(torch.float8_e8m0fnu).double()
        x = x.unflatten(1, (rows // case["block"], case["block"])) * s[:, :, None, :, None]
        seqs.append(x.reshape(-1, case["hk"], case["d"])[:n])
    return seqs


def _exact_attend(st, lens):
    case, outs, first = st["case"], [], 0
    group = case["h"] // case["hk"]
    q_all = st["q"].double().reshape(-1, case["h"], case["d"])
    k_all, v_all = _exact_sequences(st, "k", lens), _exact_sequences(st, "v", lens)
    for i, n in enumerate(lens):
        m = st["news"][i]
        q = q_all[first:first + m]
        first += m
        dist = torch.arange(n, device="cuda") - (torch.arange(m, device="cuda") + n - m)[:, None]   # key - query's own place
        hide = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hide |= dist > 0
        if case["window"] >= 0:
            hide |= dist < -case["window"]
        heads = []
        for j in range(case["hk"]):
            s = q[:, j * group:(j + 1) * group].transpose(0, 1).reshape(-1, case["d"]) @ k_all[i][:, j].t().contiguous() / math.sqrt(case["d"])
            s = s.view(group, m, n).masked_fill(hide, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            heads.append((p.view(-1, n) @ v_all[i][:, j].contiguous()).view(group, m, case["d"]).transpose(0, 1))
        outs.append(torch.cat(heads, 1))
    o = torch.cat(outs)
    return o if case["ragged"] else o.view(case["b"], case["sq"], case["h"], case["d"])
