"""Cases of the 8-bit K/V cache and of the per-head query/key norm with rotation.

Five operators, each with its plain form in elementary torch operations (32
bits throughout, rounded once at the end) and, where ``own`` is true, the
framework's call:

* ``write``   - K/V rows quantised into an 8-bit paged pool as they are written;
* ``gather``  - pool rows read back by slot;
* ``decode``  - attention of one query token per sequence over the 8-bit pool;
* ``prefill`` - causal attention of packed query rows over the 8-bit pool;
* ``norm``    - RMS norm of every query and key head with the rotary embedding.

The pool holds codes ``[num_slots, Hkv, D]`` (``float8_e4m3fn`` or ``int8``)
and one fp32 scale per (block, kv head), a power of two: a row's value is
code * scale. A write raises the scales of the blocks it touches to the
smallest power of two that holds every row (codes already there are rescaled);
a write that holds a block's first row starts the block's scale afresh.
"""

import random

import torch

own = False

_DT = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_FMT = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one decode step of 64 sequences, each appending a token to its tail block
        {"name": "write step 64", "op": "write", "kind": "append", "n": 64, "seqs": 64,
         "hkv": 4, "d": 128, "bs": 16, "dtype": "bfloat16", "fmt": "e4m3"},
        # a ragged chunk of three prompts, small heads, fp16 rows into int8
        {"name": "write chunk 777 int8", "op": "write", "kind": "prompt", "n": 777, "seqs": 3,
         "hkv": 2, "d": 64, "bs": 16, "dtype": "float16", "fmt": "int8"},
        # a prefill of eight long prompts written at once
        {"name": "write prompts 32768", "op": "write", "kind": "prompt", "n": 32768, "seqs": 8,
         "hkv": 4, "d": 128, "bs": 16, "dtype": "bfloat16", "fmt": "e4m3"},
        # a short history read back (a prefix handed to another consumer)
        {"name": "gather 333 int8", "op": "gather", "n": 333, "hkv": 2, "d": 64, "bs": 16,
         "dtype": "float16", "fmt": "int8"},
        # the histories of eight long sequences read back as 16-bit rows
        {"name": "gather 32768", "op": "gather", "n": 32768, "hkv": 4, "d": 128, "bs": 16,
         "dtype": "bfloat16", "fmt": "e4m3"},
        # one short sequence of the small geometry: latency counts
        {"name": "decode 1x201 int8", "op": "decode", "batch": 1, "lo": 201, "hi": 201, "h": 14,
         "hkv": 2, "d": 64, "bs": 16, "dtype": "float16", "fmt": "int8"},
        # the decode benchmark's batch: 64 sequences of 512 to 4096 tokens
        {"name": "decode 64x4096", "op": "decode", "batch": 64, "lo": 512, "hi": 4096, "h": 28,
         "hkv": 4, "d": 128, "bs": 16, "dtype": "bfloat16", "fmt": "e4m3"},
        # four long contexts: each split over many SMs
        {"name": "decode 4x32768 int8", "op": "decode", "batch": 4, "lo": 32768, "hi": 32768,
         "h": 28, "hkv": 4, "d": 128, "bs": 16, "dtype": "bfloat16", "fmt": "int8"},
        # a mixed step: a chunk of a prompt, a short prompt and decode rows
        {"name": "prefill mixed", "op": "prefill", "seqs": 6, "q_lo": 1, "q_hi": 300, "c_lo": 0,
         "c_hi": 700, "h": 28, "hkv": 4, "d": 128, "bs": 16, "dtype": "bfloat16", "fmt": "e4m3"},
        # four prompts of 2048 tokens after a cached prefix
        {"name": "prefill 4x2048", "op": "prefill", "seqs": 4, "q_lo": 2048, "q_hi": 2048,
         "c_lo": 17, "c_hi": 512, "h": 28, "hkv": 4, "d": 128, "bs": 16, "dtype": "bfloat16",
         "fmt": "e4m3"},
        # one decode step of 64 sequences
        {"name": "norm step 64", "op": "norm", "n": 64, "h": 28, "hkv": 4, "d": 128,
         "dtype": "bfloat16"},
        # the rows of eight long prompts
        {"name": "norm prompts 32768", "op": "norm", "n": 32768, "h": 28, "hkv": 4, "d": 128,
         "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["write", "write", "gather", "decode", "decode", "decode", "prefill", "norm"])
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    bs = rng.choice([8, 16, 16, 32, 64, 12])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    c = {"op": op, "hkv": hkv, "d": d, "bs": bs, "dtype": dtype,
         "fmt": rng.choice(["e4m3", "int8"])}
    if op == "write":
        n = _log(rng, 1, 32768 * 512 // (hkv * d) // (2 if dtype == "float32" else 1) // 2)
        kind = rng.choice(["append", "prompt"])
        if kind == "append":
            n = min(n, 1024)
        return {**c, "kind": kind, "n": n, "seqs": n if kind == "append" else min(n, rng.randint(1, 9))}
    if op == "gather":
        return {**c, "n": _log(rng, 1, 32768 * 512 // (hkv * d) // 2)}
    if op == "decode":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, min(32768, 131072 * 512 // (hkv * d) // 4 // batch))
        return {**c, "batch": batch, "lo": rng.randint(0, hi), "hi": hi,
                "h": hkv * rng.choice([1, 2, 4, 6, 7, 8, 11, 16])}
    if op == "prefill":
        seqs = rng.randint(1, 6)
        q_hi = _log(rng, 1, 1024)
        c_hi = _log(rng, 1, 1024)
        return {**c, "seqs": seqs, "q_lo": rng.randint(1, q_hi), "q_hi": q_hi,
                "c_lo": rng.randint(0, c_hi), "c_hi": c_hi, "h": hkv * rng.choice([1, 2, 3])}
    del c["bs"], c["fmt"]
    c["h"] = hkv * rng.choice([1, 2, 4, 7, 8])
    return {**c, "n": _log(rng, 1, 32768 * 4096 // ((c["h"] + hkv) * d) // 4)}


# ---------------------------------------------------------------- the format


def _pow2(e):
    """2^e as fp32, from its bits (e an integer tensor within the normal range)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_for(amax, fmt):
    """Smallest power of two s (at least 2^-126) with amax / s within the
    format's largest magnitude: 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6."""
    m, e = torch.frexp(amax)
    top, k = (1.75, 8) if fmt == "e4m3" else (1.984375, 6)
    e = e - 1 - k + (2 * m > top).to(e.dtype)
    return _pow2(torch.where(amax > 0, e, -126).clamp(min=-126))


def _code(x, fmt):
    """fp32 values within the format's range to codes, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _quantise_pool(x, bs, fmt):
    """Codes and scales of a whole pool of fp32 rows [num_slots, Hkv, D]."""
    s, h, d = x.shape
    b = x.view(s // bs, bs, h, d)
    scale = _scale_for(b.abs().amax(dim=(1, 3)), fmt)
    return _code(b / scale[:, None, :, None], fmt).view(s, h, d), scale


def _values(pool, scale, slots, bs):
    """fp32 rows of the slots (of any shape)."""
    return pool[slots].float() * scale[slots // bs].unsqueeze(-1)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _kv(g, n, hkv, d):
    """K and V rows: K with a few strong channels of its own per head, V plain."""
    k = torch.randn(n, hkv, d, generator=g, device="cuda")
    k *= torch.exp(0.7 * torch.randn(hkv, d, generator=g, device="cuda"))
    v = torch.randn(n, hkv, d, generator=g, device="cuda") * 0.5
    return k, v


def _lengths(n, lo, hi, salt=0):
    """n lengths of [lo, hi], the first of them hi: they belong to the case, so
    that every seed has outputs of the same shapes."""
    r = random.Random(salt * 1000003 + n * 8191 + lo * 131 + hi)
    return [hi] + [r.randint(lo, hi) for _ in range(n - 1)]


def _tables(g, lens, bs):
    """Block tables of shuffled blocks for sequences of these lengths."""
    counts = [-(-x // bs) for x in lens]
    perm = torch.randperm(sum(counts) + 3, generator=g, device="cuda")
    mb = max(max(counts), 1)
    bt = torch.zeros(len(lens), mb, dtype=torch.int64, device="cuda")
    off = 0
    for i, c in enumerate(counts):
        bt[i, :c] = perm[off:off + c]
        off += c
    return bt, sum(counts) + 3


def _spans(c):
    """Context lengths and query rows of every sequence of an attention case."""
    if c["op"] == "decode":
        return _lengths(c["batch"], c["lo"], c["hi"]), [1] * c["batch"]
    q = _lengths(c["seqs"], c["q_lo"], c["q_hi"])
    return [x + y for x, y in zip(q, _lengths(c["seqs"], c["c_lo"], c["c_hi"], salt=1))], q


def _pool_state(c, g, num_blocks):
    k, v = _kv(g, num_blocks * c["bs"], c["hkv"], c["d"])
    kp, ks = _quantise_pool(k, c["bs"], c["fmt"])
    vp, vs = _quantise_pool(v, c["bs"], c["fmt"])
    return {"kp": kp, "vp": vp, "ks": ks, "vs": vs}


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = _DT[c["dtype"]]
    op, hkv, d = c["op"], c["hkv"], c["d"]
    s = {"c": c}
    if op == "norm":
        n, h = c["n"], c["h"]
        qkv = torch.randn(n, (h + 2 * hkv) * d, generator=g, device="cuda").to(dt)
        pos = torch.randint(0, 32768, (n,), generator=g, device="cuda")
        inv = 1e6 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        f = pos.double()[:, None] * inv
        f = torch.cat((f, f), dim=-1)
        s.update(q=qkv[:, :h * d].view(n, h, d), k=qkv[:, h * d:(h + hkv) * d].view(n, hkv, d),
                 cos=f.cos().float(), sin=f.sin().float(),
                 wq=(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt),
                 wk=(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt), eps=1e-6)
        return s
    bs = c["bs"]
    if op == "write":
        n, m = c["n"], c["seqs"]
        if c["kind"] == "append":   # each sequence's next token, anywhere in its tail block
            lens = [x + 1 for x in _lengths(m, 0, 4 * bs)]
            new = [1] * m
        else:                       # prompts that share n rows, after a cached prefix
            ends = sorted(random.Random(n).sample(range(1, n), m - 1)) + [n]
            new = [b - a for a, b in zip([0] + ends[:-1], ends)]
            lens = [x + y for x, y in zip(new, _lengths(m, 0, 2 * bs))]
        bt, nb = _tables(g, lens, bs)
        seq = torch.tensor([i for i, x in enumerate(new) for _ in range(x)], device="cuda")
        pos = torch.tensor([p for x, y in zip(lens, new) for p in range(x - y, x)], device="cuda")
        s.update(_pool_state(c, g, nb))
        k, v = _kv(g, n, hkv, d)
        s.update(k=(k * 1.2).to(dt), v=v.to(dt), slots=bt[seq, pos // bs] * bs + pos % bs)
        return s
    if op == "gather":
        n = c["n"]
        bt, nb = _tables(g, [n], bs)
        pos = torch.arange(n, device="cuda")
        s.update(_pool_state(c, g, nb), slots=bt[0, pos // bs] * bs + pos % bs)
        return s
    lens, q_lens = _spans(c)
    rows = sum(q_lens)
    bt, nb = _tables(g, lens, bs)
    s.update(_pool_state(c, g, nb), bt=bt.to(torch.int32), max_len=max(lens),
             ctx=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             q=torch.randn(rows, c["h"], d, generator=g, device="cuda").to(dt), scale=d ** -0.5)
    if op == "prefill":
        s["max_q"] = max(q_lens)
        s["q_start"] = torch.tensor([0] + q_lens, device="cuda").cumsum(0).to(torch.int32)
    return s


# ---------------------------------------------------------------- plain forms


def _plain_write_one(rows, slots, pool, scale, bs, fmt):
    """pool and scale with the fp32 rows written at the slots."""
    touched, which = torch.unique(slots // bs, return_inverse=True)
    need = _scale_for(rows.abs().amax(dim=-1), fmt)
    new = torch.zeros(touched.numel(), rows.shape[1], device=rows.device)
    new.index_reduce_(0, which, need, "amax")
    first = torch.zeros(touched.numel(), 1, device=rows.device)
    first.index_reduce_(0, which, (slots % bs == 0).float().unsqueeze(1), "amax")
    old = scale[touched]
    now = torch.where(first > 0, new, torch.maximum(old, new))
    ratio = torch.where(first > 0, torch.ones_like(old), old / now)
    blocks = pool.view(-1, bs, *pool.shape[1:])
    blocks[touched] = _code(blocks[touched].float() * ratio[:, None, :, None], fmt)
    pool[slots] = _code(rows / now[which].unsqueeze(-1), fmt)
    scale[touched] = now


def _plain_attend(qf, kf, vf, allowed, scale):
    """qf [S, Q, H, D], kf/vf [S, T, Hkv, D], allowed [S, Q, T] -> [S, Q, H, D];
    rows with nothing allowed are zero."""
    s, n, h, d = qf.shape
    hkv = kf.shape[2]
    qg = qf.view(s, n, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(s, hkv, -1, d)
    sc = torch.matmul(qg, kf.permute(0, 2, 3, 1)).view(s, hkv, h // hkv, n, -1) * scale
    sc = sc.masked_fill(~allowed[:, None, None], float("-inf"))
    top = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del sc
    o = torch.matmul(p.view(s, hkv, -1, p.shape[-1]), vf.permute(0, 2, 1, 3))
    o = o.view(s, hkv, h // hkv, n, d) / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(s, n, h, d)


def _history(s):
    """fp32 K and V [S, max_len, Hkv, D] of every sequence, and the positions."""
    bs = s["c"]["bs"]
    pos = torch.arange(s["max_len"], device="cuda")
    slots = s["bt"].long()[:, pos // bs] * bs + pos % bs
    return _values(s["kp"], s["ks"], slots, bs), _values(s["vp"], s["vs"], slots, bs), pos


def _norm_rope(x, w, cos, sin, eps):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + eps) * w.float()
    half = y.shape[-1] // 2
    turned = torch.cat((-y[..., half:], y[..., :half]), dim=-1)
    return (y * cos.unsqueeze(1) + turned * sin.unsqueeze(1)).to(x.dtype)


def _plain(s):
    c = s["c"]
    op = c["op"]
    if op == "norm":
        return {"q": _norm_rope(s["q"], s["wq"], s["cos"], s["sin"], s["eps"]),
                "k": _norm_rope(s["k"], s["wk"], s["cos"], s["sin"], s["eps"])}
    bs, fmt = c["bs"], c["fmt"]
    dt = _DT[c["dtype"]]
    if op == "write":
        _plain_write_one(s["k"].float(), s["slots"], s["kp"], s["ks"], bs, fmt)
        _plain_write_one(s["v"].float(), s["slots"], s["vp"], s["vs"], bs, fmt)
        return {"k": s["kp"], "v": s["vp"], "ks": s["ks"], "vs": s["vs"]}
    if op == "gather":
        top = torch.finfo(dt).max
        return {"k": _values(s["kp"], s["ks"], s["slots"], bs).clamp(-top, top).to(dt),
                "v": _values(s["vp"], s["vs"], s["slots"], bs).clamp(-top, top).to(dt)}
    kf, vf, pos = _history(s)
    ctx = s["ctx"].long()
    if op == "decode":
        allowed = (pos[None] < ctx[:, None])[:, None]
        return _plain_attend(s["q"].float()[:, None], kf, vf, allowed, s["scale"])[:, 0].to(dt)
    start = s["q_start"].long()
    n = start[1:] - start[:-1]
    i = torch.arange(s["max_q"], device="cuda")
    row = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    at = (ctx - n)[:, None] + i   # position of each padded query row
    allowed = (pos <= at[..., None]) & (i < n[:, None])[..., None]
    out = _plain_attend(s["q"].float()[row], kf, vf, allowed, s["scale"])
    t = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start[1:], t, right=True)
    return out[seq, t - start[seq]].to(dt)


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    import infrared_b200 as irb

    c = s["c"]
    op = c["op"]
    if op == "norm":
        q, k = irb.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["eps"])
        return {"q": q, "k": k}
    bs = c["bs"]
    if op == "write":
        irb.cache_write_q8(s["k"], s["v"], s["kp"], s["vp"], s["ks"], s["vs"], s["slots"], bs)
        return {"k": s["kp"], "v": s["vp"], "ks": s["ks"], "vs": s["vs"]}
    if op == "gather":
        return {"k": irb.cache_gather_q8(s["kp"], s["ks"], s["slots"], bs, _DT[c["dtype"]]),
                "v": irb.cache_gather_q8(s["vp"], s["vs"], s["slots"], bs, _DT[c["dtype"]])}
    if op == "decode":
        return irb.paged_decode_q8(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["bt"], s["ctx"],
                                   s["scale"], bs)
    return irb.paged_prefill_q8(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["bt"], s["ctx"],
                                s["q_start"], s["scale"], bs)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- work


def work(case):
    c = case
    e = 4 if c["dtype"] == "float32" else 2
    row = c["hkv"] * c["d"]
    if c["op"] == "norm":
        rows = c["n"] * (c["h"] + c["hkv"]) * c["d"]
        return {"bytes": 2 * rows * e + c["n"] * c["d"] * 8, "flops": 8 * rows}
    if c["op"] == "write":
        return {"bytes": 2 * c["n"] * row * (e + 1) + 8 * c["n"], "flops": 4 * c["n"] * row}
    if c["op"] == "gather":
        return {"bytes": 2 * c["n"] * row * (e + 1) + 8 * c["n"], "flops": 2 * c["n"] * row}
    lens, q_lens = _spans(c)
    pairs = sum(n * (x - n) + n * (n + 1) // 2 for x, n in zip(lens, q_lens))
    return {"bytes": 2 * sum(lens) * row + 2 * sum(q_lens) * c["h"] * c["d"] * e,
            "flops": 4 * pairs * c["h"] * c["d"]}


# ---------------------------------------------------------------- 64 bits


def _two_to(e):
    """2^e in fp64, from its bits (e holds whole numbers)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_scale(amax, fmt):
    """As fp64: 2^ceil(log2(amax / largest)), the logarithm's last step settled
    by comparing, at least 2^-126."""
    top = 448.0 if fmt == "e4m3" else 127.0
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / top))
    e = e + (_two_to(e) * top < amax).double() - (_two_to(e - 1) * top >= amax).double()
    return _two_to(e.clamp(min=-126))


def _exact_code(x, fmt):
    """The nearest value of the format, ties to even, in fp64."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -60))).clamp(min=-6)
    e = e + (_two_to(e + 1) <= x.abs()).double() - ((_two_to(e) > x.abs()) & (e > -6)).double()
    step = _two_to(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_write(rows, slots, pool, scale, bs, fmt):
    """The pool's codes and scales after the write, in fp64: the blocks laid out
    whole, with a mark at each row that the write brings."""
    nb, h, d = scale.shape[0], pool.shape[1], pool.shape[2]
    mark = torch.zeros(nb * bs, dtype=torch.bool, device="cuda")
    mark[slots] = True
    fresh = torch.zeros(nb * bs, h, d, dtype=torch.float64, device="cuda")
    fresh[slots] = rows.double()
    fresh, mark = fresh.view(nb, bs, h, d), mark.view(nb, bs)
    codes = pool.double().view(nb, bs, h, d)
    old = scale.double()
    hit, begun = mark.any(dim=1)[:, None], mark[:, 0][:, None]
    need = _exact_scale(fresh.abs().amax(dim=(1, 3)), fmt)
    now = torch.where(begun, need, torch.where(hit, torch.maximum(old, need), old))
    kept = torch.where(begun[..., None, None], codes, _exact_code(codes * (old / now)[:, None, :, None], fmt))
    out = torch.where(mark[..., None, None], _exact_code(fresh / now[:, None, :, None], fmt), kept)
    return out.view(nb * bs, h, d), now


def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    if op == "norm":
        out = {}
        cs, sn = s["cos"].double()[:, None], s["sin"].double()[:, None]
        for name, w in (("q", s["wq"]), ("k", s["wk"])):
            x = s[name].double()
            y = x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / c["d"] + s["eps"]) * w.double()
            a, b = y.chunk(2, dim=-1)
            ca, cb = cs.chunk(2, dim=-1)
            sa, sb = sn.chunk(2, dim=-1)
            out[name] = torch.cat((a * ca - b * sa, b * cb + a * sb), dim=-1)
        return out
    bs, fmt = c["bs"], c["fmt"]
    if op == "write":
        k, ks = _exact_write(s["k"], s["slots"], s["kp"], s["ks"], bs, fmt)
        v, vs = _exact_write(s["v"], s["slots"], s["vp"], s["vs"], bs, fmt)
        whole = fmt == "int8"   # whole numbers: held to equality with the plain form's
        return {"k": None if whole else k, "v": None if whole else v, "ks": ks, "vs": vs}
    if op == "gather":
        top = torch.finfo(_DT[c["dtype"]]).max
        at = s["slots"] // bs
        return {"k": (s["kp"][s["slots"]].double() * s["ks"].double()[at][..., None]).clamp(-top, top),
                "v": (s["vp"][s["slots"]].double() * s["vs"].double()[at][..., None]).clamp(-top, top)}
    rep = c["h"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens = s["ctx"].tolist()
    starts = s["q_start"].tolist() if op == "prefill" else list(range(len(lens) + 1))
    for i, n in enumerate(lens):
        lo, hi = starts[i], starts[i + 1]
        if n == 0:
            continue
        p = torch.arange(n, device="cuda")
        sl = s["bt"][i].long()[p // bs] * bs + p % bs
        k = s["kp"][sl].double() * s["ks"].double()[sl // bs][..., None]
        v = s["vp"][sl].double() * s["vs"].double()[sl // bs][..., None]
        row = torch.arange(n - (hi - lo), n, device="cuda")
        for h in range(c["h"]):
            w = s["q"][lo:hi, h].double() @ k[:, h // rep].T * s["scale"]
            w = torch.softmax(w.masked_fill(p[None] > row[:, None], float("-inf")), dim=-1)
            out[lo:hi, h] = w @ v[:, h // rep]
    return out
