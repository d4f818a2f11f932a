"""8-bit K/V cache and its attention on the GPU against the fp64 restatement.

Codes, scales and rows read back are exact (a power-of-two scale divides
exactly, so a code has one rounding, the same everywhere). Attention is held
to bounds counted from the roundings of each kernel, row by row:

* a score is a sum of D products accumulated in fp32: at most D steps of
  2^-23 (a tensor core may truncate) of sum_d |q_d k_d|, plus a few roundings
  of the score itself (scaling, exponent's argument);
* a relative error e of every weight moves the output by at most 2 e times
  sum_j p_j |v_j| (numerator and denominator);
* weights rounded to fp16 (16-bit q): 2^-11 each, 2^-24 of 2^-7 below the
  normal range; sums over T tokens in fp32: T steps of 2^-23 at most;
* the exponential instruction: 2^-22;
* the output rounding: half a unit of the output type.
"""

import numpy as np
import pytest
import torch

import infrared_b200 as irb
from infrared_b200 import ops
from infrared_b200 import workloads as wl
from oracle import kv_q8_np as q8

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda"
FMT = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@pytest.fixture(autouse=True)
def _clean_errors():
    ops.error_flag().zero_()
    yield
    ops.check_device_errors()


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().double().cpu().numpy()


def codes_to(codes, fmt):
    return dev(codes.astype(np.float32)).to(FMT[fmt])


def make_pool(rng, nb, bs, hkv, d, fmt, spread=1.0):
    """Codes and scales of a random pool, one (block, head) quantised at a time."""
    codes, scale = np.zeros((nb * bs, hkv, d)), np.zeros((nb, hkv))
    rows = rng.normal(size=(nb * bs, hkv, d)) * spread * \
        np.exp(rng.normal(size=(nb, 1, hkv, 1)) * np.ones((nb, bs, hkv, 1))).reshape(nb * bs, hkv, 1)
    q8.write(codes, scale, rows, range(nb * bs), bs, fmt)
    return codes, scale


# ---------------------------------------------------------------- cache write


def _write_case(rng, n, hkv, d, bs, nb, fmt, dtype, order="mixed"):
    codes, scale = make_pool(rng, nb, bs, hkv, d, fmt, 0.2)
    rows = [dev(rng.normal(size=(n, hkv, d)) * np.exp(rng.normal(size=(n, hkv, 1)))).to(dtype)
            for _ in range(2)]
    slots = rng.permutation(nb * bs)[:n]
    if order == "runs":
        slots = np.sort(slots)
    return codes, scale, rows, slots


def _check_write(codes, scale, rows, slots, bs, fmt, neg=()):
    slots = np.array(slots, np.int64)
    slots[list(neg)] = -1
    kp, vp = codes_to(codes, fmt), codes_to(codes, fmt)
    ks, vs = dev(scale.astype(np.float32)), dev(scale.astype(np.float32))
    irb.cache_write_q8(rows[0], rows[1], kp, vp, ks, vs, dev(slots), bs)
    for pool, sc, x in ((kp, ks, rows[0]), (vp, vs, rows[1])):
        want, ws = codes.copy(), scale.copy()
        q8.write(want, ws, host(x), slots, bs, fmt)
        np.testing.assert_array_equal(host(sc), ws)
        np.testing.assert_array_equal(host(pool), want)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,hkv,d,bs,nb", [
    (1, 1, 64, 16, 3), (1, 4, 128, 1, 5), (5, 2, 64, 5, 4), (64, 4, 128, 16, 80),
    (333, 2, 64, 16, 40), (100, 8, 128, 8, 60), (70, 3, 128, 64, 4), (40, 1, 128, 1024, 1),
])
def test_write(n, hkv, d, bs, nb, dtype, fmt):
    rng = np.random.default_rng(n * 7 + d + bs)
    _check_write(*_write_case(rng, n, hkv, d, bs, nb, fmt, dtype), bs, fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("n,hkv,d,bs,nb", [
    (1024, 2, 64, 16, 100), (1025, 2, 64, 16, 100), (3000, 1, 128, 16, 200), (2500, 2, 64, 12, 250),
    (1500, 1, 64, 1, 1600), (1030, 2, 64, 256, 5),
])
def test_write_many_tokens(n, hkv, d, bs, nb, order, fmt):
    rng = np.random.default_rng(n + bs)
    case = _write_case(rng, n, hkv, d, bs, nb, fmt, torch.bfloat16, order)
    _check_write(*case, bs, fmt, neg=(0, 17, n - 1))


@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("n,bs,nb", [(8193, 16, 600), (20000, 16, 1400), (32769, 16, 2100),
                                     (20000, 1, 30000)])
def test_write_links_of_long_calls(n, bs, nb, order):
    """Calls whose rows are linked per block, over many CTAs and blocks."""
    rng = np.random.default_rng(n)
    case = _write_case(rng, n, 1, 64, bs, nb, "e4m3", torch.bfloat16, order)
    _check_write(*case, bs, "e4m3", neg=(0, 17, n - 1))


@pytest.mark.parametrize("n", [40, 1100])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_same_slot_twice_keeps_the_last_row(fmt, n):
    rng = np.random.default_rng(n)
    codes, scale, rows, slots = _write_case(rng, n, 2, 64, 16, 80, fmt, torch.float16)
    slots[n // 2:] = slots[:n - n // 2]
    _check_write(codes, scale, rows, slots, 16, fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_step_by_step_equals_the_restatement(fmt):
    """A prompt, then tokens that raise the tail block's scale, on row views of
    one projection output."""
    rng = np.random.default_rng(8)
    hkv, d, bs, nb = 2, 64, 16, 4
    codes, scale = make_pool(rng, nb, bs, hkv, d, fmt)
    kp, vp = codes_to(codes, fmt), codes_to(codes, fmt)
    ks, vs = dev(scale.astype(np.float32)), dev(scale.astype(np.float32))
    wk, wv, sk, sv = codes.copy(), codes.copy(), scale.copy(), scale.copy()
    table, pos = [2, 0, 3], 0
    for n, size in ((19, 1.0), (1, 0.5), (1, 3.0), (1, 40.0), (9, 0.1), (3, 9.0), (1, 1e-3)):
        x = dev(rng.normal(size=(n, 3 * hkv * d)) * size).to(torch.bfloat16)
        k, v = x[:, hkv * d:2 * hkv * d], x[:, 2 * hkv * d:]
        p = np.arange(pos, pos + n)
        slots = np.array(table)[p // bs] * bs + p % bs
        irb.cache_write_q8(k.view(n, hkv, d), v.view(n, hkv, d), kp, vp, ks, vs, dev(slots), bs)
        q8.write(wk, sk, host(k).reshape(n, hkv, d), slots, bs, fmt)
        q8.write(wv, sv, host(v).reshape(n, hkv, d), slots, bs, fmt)
        pos += n
    for got, want in ((kp, wk), (vp, wv), (ks, sk), (vs, sv)):
        np.testing.assert_array_equal(host(got), want)


@pytest.mark.parametrize("offset", [0, 1, 3])
def test_write_unaligned_rows(offset):
    rng = np.random.default_rng(5)
    n, hkv, d, bs = 20, 2, 64, 16
    codes, scale, _, slots = _write_case(rng, n, hkv, d, bs, 4, "e4m3", torch.bfloat16)
    rows = []
    for _ in range(2):
        flat = dev(rng.normal(size=n * (hkv * d + 5) + 8)).to(torch.bfloat16)
        rows.append(flat[offset:].as_strided((n, hkv, d), (hkv * d + 5, d, 1),
                                             flat.storage_offset() + offset))
    _check_write(codes, scale, rows, slots, bs, "e4m3")


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_values_that_are_not_finite(fmt):
    rng = np.random.default_rng(6)
    codes, scale, rows, _ = _write_case(rng, 6, 2, 64, 16, 3, fmt, torch.float32)
    rows[0][1, 0, 5] = float("nan")
    rows[0][2, 1, 7] = float("inf")
    rows[1][3, 0, 0] = float("-inf")
    rows[1][4] = 0.0
    rows[1][5] = 1e-42
    slots = np.array([16, 17, 18, 35, 36, 37])
    _check_write(codes, scale, rows, slots, 16, fmt)
    # a NaN scale of an int8 block stays until the block is begun again
    scale[2, 0] = np.nan if fmt == "int8" else scale[2, 0]
    _check_write(codes, scale, rows, np.array([33, 34, 35, 36, 37, 38]), 16, fmt)
    _check_write(codes, scale, rows, np.array([33, 34, 32, 36, 37, 38]), 16, fmt)


@pytest.mark.parametrize("n", [5, 1200])
def test_write_slot_outside_the_pool_is_flagged_and_skipped(n):
    rng = np.random.default_rng(9)
    codes, scale, rows, slots = _write_case(rng, n, 1, 64, 16, 90, "e4m3", torch.bfloat16)
    bad = slots.copy()
    bad[3] = 90 * 16
    kp, vp = codes_to(codes, "e4m3"), codes_to(codes, "e4m3")
    ks, vs = dev(scale.astype(np.float32)), dev(scale.astype(np.float32))
    irb.cache_write_q8(rows[0], rows[1], kp, vp, ks, vs, dev(bad.astype(np.int64)), 16)
    with pytest.raises(irb.DeviceError, match="SLOT"):
        irb.check_device_errors()
    want, ws = codes.copy(), scale.copy()
    bad[3] = -1
    q8.write(want, ws, host(rows[0]), bad, 16, "e4m3")
    np.testing.assert_array_equal(host(kp), want)
    np.testing.assert_array_equal(host(ks), ws)


# ---------------------------------------------------------------- gather


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gather(fmt, dtype):
    rng = np.random.default_rng(1)
    for hkv, d, bs, nb in ((2, 64, 16, 20), (4, 128, 5, 9), (1, 64, 1, 7)):
        codes, scale = make_pool(rng, nb, bs, hkv, d, fmt)
        scale[0] = 2.0 ** 12   # values beyond fp16 saturate
        slots = rng.integers(0, nb * bs, size=(3, 11))
        got = irb.cache_gather_q8(codes_to(codes, fmt), dev(scale.astype(np.float32)), dev(slots),
                                  bs, dtype)
        assert got.shape == (3, 11, hkv, d) and got.dtype == dtype
        top = torch.finfo(dtype).max
        want = torch.from_numpy(q8.values(codes, scale, bs)[slots]).clamp(-top, top).to(dtype)
        assert torch.equal(got.cpu(), want)
        assert irb.cache_gather_q8(codes_to(codes, fmt), dev(scale.astype(np.float32)),
                                   dev(slots[:0]), bs, dtype).numel() == 0


def test_gather_bad_slots_give_zero_rows():
    rng = np.random.default_rng(1)
    codes, scale = make_pool(rng, 3, 16, 2, 64, "e4m3")
    got = irb.cache_gather_q8(codes_to(codes, "e4m3"), dev(scale.astype(np.float32)),
                              dev(np.array([-1, 5, 48])), 16, torch.float32)
    with pytest.raises(irb.DeviceError, match="SLOT"):
        irb.check_device_errors()
    assert not got[0].any() and not got[2].any()
    np.testing.assert_array_equal(host(got[1]), q8.values(codes, scale, 16)[5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_largest_values(dtype):
    """The largest value of the type comes back as its code does, saturated where
    the rounded code times its scale (2^128 for 32 exponents more) is beyond it."""
    top = torch.finfo(dtype).max
    for fmt in ("e4m3", "int8"):
        x = torch.full((16, 1, 64), top, dtype=dtype, device="cuda")
        x[1] = -top
        pool = codes_to(np.zeros((16, 1, 64)), fmt)
        sc = torch.zeros(1, 1, device="cuda")
        irb.cache_write_q8(x, x, pool, pool.clone(), sc, sc.clone(), torch.arange(16, device="cuda"), 16)
        codes, scale = np.zeros((16, 1, 64)), np.zeros((1, 1))
        q8.write(codes, scale, x.double().cpu().numpy(), range(16), 16, fmt)
        assert float(sc) == scale[0, 0]
        got = irb.cache_gather_q8(pool, sc, torch.arange(16, device="cuda"), 16, dtype)
        want = torch.from_numpy(q8.values(codes, scale, 16)).clamp(-top, top).to(dtype)
        assert torch.equal(got.cpu(), want) and torch.isfinite(got).all()


# ---------------------------------------------------------------- attention


def attend_tolerance(out, weighted, size, n, d, dtype, low_p):
    """The bound of the module's header for one row."""
    e = (d + 8) * 2.0 ** -23 * size + 2.0 ** -21 + n * 2.0 ** -23
    if low_p:
        e = e + 2.0 ** -11
    tail = n * 2.0 ** -31 * np.abs(weighted).max() if low_p else 0.0
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return 2 * e[:, None] * weighted + tail + half * np.abs(out) * (1 + 2.0 ** -6) + tiny


def check_decode(w, fmt, dtype, path=None, seed=0, q=None, spread=1.0, out=None, width=0):
    rng = np.random.default_rng(seed)
    kc, ks = make_pool(rng, w.num_blocks, w.block_size, w.num_kv_heads, w.head_dim, fmt, spread)
    vc, vs = make_pool(rng, w.num_blocks, w.block_size, w.num_kv_heads, w.head_dim, fmt)
    if q is None:
        q = dev(rng.normal(size=(w.batch, w.num_heads, w.head_dim))).to(dtype)
    cols = -(-width // w.block_size) - w.block_tables.shape[1]   # tables of `width` tokens
    bt, ctx = dev(np.pad(w.block_tables, ((0, 0), (0, max(cols, 0))))), dev(w.context_lens)
    kp, vp = codes_to(kc, fmt), codes_to(vc, fmt)
    if path is not None:
        assert ops.decode_plan_q8(q, kp, bt, w.block_size)[0] == path
    got = irb.paged_decode_q8(q, kp, vp, dev(ks.astype(np.float32)), dev(vs.astype(np.float32)),
                              bt, ctx, w.scale, w.block_size, out=out)
    kv, vv = q8.values(kc, ks, w.block_size), q8.values(vc, vs, w.block_size)
    g, qh = host(got), host(q)
    for i in range(w.batch):
        n = int(w.context_lens[i])
        want, weighted, size = q8.attend(
            qh[i], q8.history(kv, w.block_tables[i], n, w.block_size),
            q8.history(vv, w.block_tables[i], n, w.block_size), w.scale)
        tol = attend_tolerance(want, weighted, size, n, w.head_dim, dtype, path == 2)
        err = np.abs(g[i] - want)
        assert (err <= tol).all(), (i, n, float((err - tol).max()), float(err.max()))
    return got


GEOM = [  # H, Hkv, D, block size, path of 16-bit q
    (28, 4, 128, 16, 2), (14, 2, 64, 16, 2), (8, 8, 128, 32, 2), (16, 8, 64, 48, 2),
    (8, 1, 128, 16, 2), (3, 3, 64, 16, 2), (11, 1, 128, 16, 2), (32, 2, 64, 16, 2),
    (44, 4, 128, 64, 2), (28, 4, 128, 8, 2), (14, 2, 64, 8, 2), (12, 1, 64, 8, 2),
    (128, 8, 128, 16, 2), (6, 6, 128, 8, 2), (28, 4, 128, 12, 1), (14, 2, 64, 5, 1),
    (4, 2, 64, 1, 1),
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("geom", GEOM)
def test_decode_bf16(geom, fmt):
    h, hkv, d, bs, path = geom
    w = wl.custom(h + bs, 7, h, hkv, d, bs, 0, 150)
    w.context_lens[:4] = [0, 1, 150, 17]
    check_decode(w, fmt, torch.bfloat16, path)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("geom", GEOM)
def test_decode_wide_tables(geom, fmt):
    """The same in equal shares of all tokens (tables wider than the contexts)."""
    h, hkv, d, bs, path = geom
    w = wl.custom(h + bs, 7, h, hkv, d, bs, 0, 150)
    w.context_lens[:4] = [0, 1, 150, 17]
    check_decode(w, fmt, torch.bfloat16, path, width=2000)


@pytest.mark.parametrize("geom", GEOM[:14])
def test_decode_whole_sequences(geom):
    """A CTA per sequence: none of its results goes through the merge, so a row does
    not depend on the others."""
    h, hkv, d, bs, path = geom
    w = _with_lengths(5, [500, 0, 1, 16, 17, 256, 257, 33, 129, 400], h, hkv, d, bs)
    got = check_decode(w, "e4m3", torch.bfloat16, path)
    rng = np.random.default_rng(0)
    kc, ks = make_pool(rng, w.num_blocks, bs, hkv, d, "e4m3")
    vc, vs = make_pool(rng, w.num_blocks, bs, hkv, d, "e4m3")
    q = dev(rng.normal(size=(w.batch, h, d))).to(torch.bfloat16)
    for i in (0, 1, 6):
        one = irb.paged_decode_q8(q[i:i + 1], codes_to(kc, "e4m3"), codes_to(vc, "e4m3"),
                                  dev(ks.astype(np.float32)), dev(vs.astype(np.float32)),
                                  dev(w.block_tables[i:i + 1]), dev(w.context_lens[i:i + 1]),
                                  w.scale, bs)
        if 10 * hkv <= 148:   # (else ten sequences take more heads a CTA than one)
            assert torch.equal(one[0], got[i])
    bad = w.context_lens.copy()
    bad[0], bad[3] = -1, w.block_tables.shape[1] * bs + 1   # read as none and as all
    bt = w.block_tables.copy()
    bt[5, 0] = w.num_blocks
    irb.paged_decode_q8(q, codes_to(kc, "e4m3"), codes_to(vc, "e4m3"),
                        dev(ks.astype(np.float32)), dev(vs.astype(np.float32)), dev(bt), dev(bad),
                        w.scale, bs)
    with pytest.raises(irb.DeviceError, match="CONTEXT_LEN"):
        irb.check_device_errors()


def _with_lengths(seed, lens, h, hkv, d, bs):
    """A workload of exactly these context lengths."""
    rng = np.random.default_rng(seed)
    ctx = np.array(lens, np.int32)
    nb = int(((ctx.astype(np.int64) + bs - 1) // bs).sum()) + 3
    bt, _ = wl.assign_blocks(rng, ctx, bs, nb)
    return wl.Workload("lens", len(lens), h, hkv, d, bs, nb, "bfloat16", d ** -0.5, 1.0, ctx, bt,
                       wl.tail_slots(bt, ctx, bs))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("geom", [GEOM[0], GEOM[1], GEOM[6], GEOM[9], GEOM[15]])
def test_decode_other_types(geom, dtype, fmt):
    h, hkv, d, bs, path = geom
    w = _with_lengths(3, [1, 16, 0, 33, 129, 8], h, hkv, d, bs)
    check_decode(w, fmt, dtype, path if dtype == torch.float16 else 1, spread=3.0)


@pytest.mark.parametrize("lens", [
    [1], [0], [0, 0, 0], [5000], [2047, 2048, 2049], [15, 16, 17, 31, 32, 33] * 4,
    [1] * 300, [7, 0] * 150, [1500, 3, 0, 800] * 5,
])
def test_decode_lengths(lens):
    """One sequence over all SMs, many short ones in one CTA, empty rows between."""
    h, hkv, d = (28, 4, 128) if sum(lens) < 3000 else (8, 2, 64)
    check_decode(_with_lengths(len(lens), lens, h, hkv, d, 16), "e4m3", torch.bfloat16, 2)


@pytest.mark.parametrize("hkv", [1, 2, 4, 8])
@pytest.mark.parametrize("rep", [1, 8, 9, 16])
@pytest.mark.parametrize("width", [0, 2000])
def test_decode_head_groups(hkv, rep, width):
    w = _with_lengths(hkv, [300, 1, 77, 200], hkv * rep, hkv, 128, 16)
    check_decode(w, "int8", torch.bfloat16, 2, width=width)


@pytest.mark.parametrize("batch", [30, 60, 140])
def test_decode_whole_sequences_of_several_heads(batch):
    """2, 4 and 8 heads a CTA: as many as leave the CTAs in one wave."""
    rng = np.random.default_rng(batch)
    w = _with_lengths(batch, rng.integers(0, 300, batch).tolist(), 16, 8, 64, 16)
    check_decode(w, "e4m3", torch.bfloat16, 2)


def test_decode_strided_and_unaligned_rows():
    w = _with_lengths(2, [40, 100, 3], 14, 2, 64, 16)
    rng = np.random.default_rng(4)
    flat = dev(rng.normal(size=3 * 2000 + 16)).to(torch.bfloat16)
    for off, stride in ((0, 2000), (1, 901), (4, 1000), (0, 904)):
        q = flat[off:].as_strided((3, 14, 64), (stride, 64, 1), off)
        check_decode(w, "e4m3", torch.bfloat16, 2, q=q)
    out = torch.full((3, 14 * 64 + 8), 9.0, dtype=torch.bfloat16, device=DEV)
    check_decode(w, "e4m3", torch.bfloat16, 2, out=out[:, :14 * 64].view(3, 14, 64))
    assert (out[:, 14 * 64:] == 9.0).all()
    # rows of out that do not start on 16 bytes take the CUDA-core kernel
    odd = torch.empty(3 * (14 * 64 + 1), dtype=torch.bfloat16, device=DEV)
    check_decode(w, "e4m3", torch.bfloat16, None, out=odd.as_strided((3, 14, 64), (897, 64, 1)))


def test_decode_large_and_small_queries():
    """q far outside fp16's range, and rows of zeros."""
    w = _with_lengths(2, [40, 100, 3], 14, 2, 64, 16)
    rng = np.random.default_rng(4)
    for size in (1e-30, 1e-8, 30.0):
        q = dev(rng.normal(size=(3, 14, 64)) * size).to(torch.bfloat16)
        q[1, 3] = 0.0
        check_decode(w, "e4m3", torch.bfloat16, 2, q=q)
    # the same scores from a huge q and a tiny softmax scale
    w.scale = 1e-25
    check_decode(w, "int8", torch.bfloat16, 2, q=dev(rng.normal(size=(3, 14, 64)) * 1e24).to(torch.bfloat16))


@pytest.mark.parametrize("fmt,dtype,bs", [
    ("e4m3", torch.bfloat16, 16), ("e4m3", torch.bfloat16, 8), ("e4m3", torch.float32, 16),
    ("int8", torch.bfloat16, 16), ("int8", torch.bfloat16, 8), ("int8", torch.float32, 5)])
def test_decode_garbage_past_the_context(fmt, dtype, bs):
    """NaN codes and scales in rows and blocks that no sequence reaches change nothing."""
    w = _with_lengths(5, [17, 1, 40, 9, 0], 14, 2, 64, bs)
    rng = np.random.default_rng(2)
    kc, ks = make_pool(rng, w.num_blocks, bs, 2, 64, fmt)
    q = dev(rng.normal(size=(5, 14, 64))).to(dtype)
    used = np.zeros(w.num_blocks * bs, bool)
    held = np.zeros(w.num_blocks, bool)
    for i, n in enumerate(w.context_lens):
        p = np.arange(n)
        used[w.block_tables[i, p // bs] * bs + p % bs] = True
        held[w.block_tables[i, p // bs]] = True
    bt, ctx = dev(w.block_tables), dev(w.context_lens)

    def run(codes, scale):
        pool, sc = codes_to(codes, fmt), dev(scale.astype(np.float32))
        return irb.paged_decode_q8(q, pool, pool, sc, sc, bt, ctx, w.scale, bs)

    clean = run(kc, ks)
    dirty, dsc = kc.copy(), ks.copy()
    dirty[~used] = np.nan if fmt == "e4m3" else 127
    dsc[~held] = np.nan
    assert torch.equal(run(dirty, dsc), clean)
    assert not clean[4].any()


@pytest.mark.parametrize("dtype,bs", [(torch.bfloat16, 16), (torch.float32, 16)])
def test_decode_nan_in_the_history_reaches_the_row(dtype, bs):
    w = _with_lengths(5, [17, 1, 300], 14, 2, 64, bs)
    rng = np.random.default_rng(2)
    kc, ks = make_pool(rng, w.num_blocks, bs, 2, 64, "e4m3")
    vc, vs = make_pool(rng, w.num_blocks, bs, 2, 64, "e4m3")
    q = dev(rng.normal(size=(3, 14, 64))).to(dtype)
    kc[w.block_tables[1, 0] * bs, 0, 3] = np.nan          # the only key of row 1, head group 0
    vc[w.block_tables[2, 2] * bs + 1, 1, 9] = np.nan       # one element of V
    out = irb.paged_decode_q8(q, codes_to(kc, "e4m3"), codes_to(vc, "e4m3"),
                              dev(ks.astype(np.float32)), dev(vs.astype(np.float32)),
                              dev(w.block_tables), dev(w.context_lens), w.scale, bs)
    bad = torch.isnan(out).cpu()
    want = torch.zeros_like(bad)
    want[1, :7] = True
    want[2, 7:, 9] = True
    assert torch.equal(bad, want)


def test_decode_scales_of_any_value():
    """Scales that are no powers of two, and very different ones in one sequence."""
    w = _with_lengths(5, [60, 33], 14, 2, 64, 16)
    rng = np.random.default_rng(2)
    for fmt, bs in (("int8", 16), ("e4m3", 8)):
        w = _with_lengths(5, [60, 33], 14, 2, 64, bs)
        kc, _ = make_pool(rng, w.num_blocks, bs, 2, 64, fmt)
        ks = np.float32(rng.uniform(0.001, 0.01, size=(w.num_blocks, 2)))
        vs = np.float32(np.exp(rng.normal(size=(w.num_blocks, 2)) * 8))
        q = dev(rng.normal(size=(2, 14, 64))).to(torch.float16)
        got = host(irb.paged_decode_q8(q, codes_to(kc, fmt), codes_to(kc, fmt), dev(ks), dev(vs),
                                       dev(w.block_tables), dev(w.context_lens), w.scale, bs))
        kv, vv = q8.values(kc, ks, bs), q8.values(kc, vs, bs)
        for i, n in enumerate(w.context_lens):
            want, weighted, size = q8.attend(host(q[i]), q8.history(kv, w.block_tables[i], n, bs),
                                             q8.history(vv, w.block_tables[i], n, bs), w.scale)
            tol = attend_tolerance(want, weighted, size, n, 64, torch.float16, True)
            sure = np.abs(want) < 6e4   # fp16 outputs beyond its range are infinite
            assert (np.abs(got[i] - want)[sure] <= tol[sure]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_bad_block_ids_are_flagged(dtype):
    w = _with_lengths(5, [60, 33], 14, 2, 64, 16)
    rng = np.random.default_rng(2)
    kc, ks = make_pool(rng, w.num_blocks, 16, 2, 64, "e4m3")
    bt = w.block_tables.copy()
    bt[0, 1], bt[0, 2] = -5, w.num_blocks
    q = dev(rng.normal(size=(2, 14, 64))).to(dtype)
    sc, pool = dev(ks.astype(np.float32)), codes_to(kc, "e4m3")
    out = irb.paged_decode_q8(q, pool, pool, sc, sc, dev(bt), dev(w.context_lens), w.scale, 16)
    with pytest.raises(irb.DeviceError, match="BLOCK_ID"):
        irb.check_device_errors()
    good = irb.paged_decode_q8(q, pool, pool, sc, sc, dev(w.block_tables), dev(w.context_lens),
                               w.scale, 16)
    # the other sequence is untouched (its pieces may be cut alike: same lengths)
    assert torch.equal(out[1], good[1])


def test_decode_is_deterministic_and_replays():
    w = _with_lengths(9, [700, 33, 1200, 5], 28, 4, 128, 16)
    rng = np.random.default_rng(2)
    kc, ks = make_pool(rng, w.num_blocks, 16, 4, 128, "e4m3")
    pool, sc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32))
    bt, ctx = dev(w.block_tables), dev(w.context_lens)
    q = dev(rng.normal(size=(4, 28, 128))).to(torch.bfloat16)
    q2 = dev(rng.normal(size=(4, 28, 128))).to(torch.bfloat16)
    call = lambda x, out=None: irb.paged_decode_q8(x, pool, pool, sc, sc, bt, ctx, w.scale, 16,  # noqa: E731
                                                   out=out)
    first, second = call(q), call(q2)
    assert torch.equal(call(q), first)
    out1, out2 = torch.empty_like(q), torch.empty_like(q)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        call(q, out1)
    with torch.cuda.graph(g2):
        call(q2, out2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):   # two replayed graphs at once: neither shares scratch
        g1.replay()
        with torch.cuda.stream(side):
            g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(out1, first) and torch.equal(out2, second)


# ---------------------------------------------------------------- prefill


def check_prefill(h, hkv, d, bs, spans, dtype, fmt, path, q=None, out=None, width=0, spread=1.0,
                  dirty=False, more=0):
    """Every row of a packed frame against 64 bits; `width`: extra table columns;
    `more`: rows of no sequence behind the others (a frame of many rows);
    `dirty`: NaN in the workspace and in pool rows that no row attends."""
    rng = np.random.default_rng(h + d)
    f = wl.prefill_frame("t", 3, [s for s, _ in spans], [n for _, n in spans], h, hkv, d, bs)
    kc, ks = make_pool(rng, f.num_blocks, bs, hkv, d, fmt, spread)
    vc, vs = make_pool(rng, f.num_blocks, bs, hkv, d, fmt)
    if q is None:
        q = dev(rng.normal(size=(f.total_q + more, h, d))).to(dtype)
    table = np.pad(f.block_tables, ((0, 0), (0, width)))
    kd, vd, ksd, vsd = kc.copy(), vc.copy(), ks.copy(), vs.copy()
    if dirty:
        used = np.zeros(f.num_blocks * bs, bool)
        for i, n in enumerate(f.context_lens):
            p = np.arange(n)
            used[f.block_tables[i, p // bs] * bs + p % bs] = True
        kd[~used] = vd[~used] = np.nan if fmt == "e4m3" else 127
    kp, vp = codes_to(kd, fmt), codes_to(vd, fmt)
    bt, ctx, qs = dev(table), dev(f.context_lens), dev(f.q_start)
    got_path, nbytes = ops.prefill_plan_q8(q, kp, bt, qs, bs)
    assert got_path == path
    ws = torch.full((max(nbytes, 256),), 0xff, dtype=torch.uint8, device=DEV) if dirty else None
    got = host(irb.paged_prefill_q8(q, kp, vp, dev(ksd.astype(np.float32)),
                                    dev(vsd.astype(np.float32)), bt, ctx, qs, f.scale, bs, out=out,
                                    ws=ws))
    kv, vv = q8.values(kc, ks, bs), q8.values(vc, vs, bs)
    low = path in (2, 3)
    half = torch.finfo(dtype).eps / 2
    for i, (start, n) in enumerate(spans):
        for r in range(0, n, 1 if n < 50 else 13):
            t = start + r + 1
            row = int(f.q_start[i]) + r
            want, weighted, size = q8.attend(host(q[row]),
                                             q8.history(kv, f.block_tables[i], t, bs),
                                             q8.history(vv, f.block_tables[i], t, bs), f.scale)
            tol = attend_tolerance(want, weighted, size, t, d, dtype, path == 1 and dtype !=
                                   torch.float32)
            if low:
                # weights rounded to the type; in fp16 a weight below 2^-14 (of a
                # largest of 1) is rounded to a multiple of 2^-24, so it is off by
                # up to 2^-25 whatever its size: t of them move sum p v / sum p,
                # whose denominator is at least 1, by up to t 2^-25 max |v|. Rows of
                # the expanded pool below fp16's normal range: 2^-25 each likewise
                tol = tol + 2 * half * weighted
                if dtype == torch.float16:
                    vmax = np.abs(q8.history(vv, f.block_tables[i], t, bs)).max()
                    tol = tol + t * 2.0 ** -25 * vmax + 2.0 ** -24
            err = np.abs(got[row] - want)
            assert (err <= tol).all(), (i, r, float((err - tol).max()))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,hkv,d,bs,spans", [
    (28, 4, 128, 16, [(0, 130), (17, 1), (50, 40)]), (14, 2, 64, 16, [(3, 5), (0, 1), (0, 200)]),
    (4, 4, 128, 12, [(20, 30), (0, 7)]), (16, 1, 64, 8, [(9, 33)]),
    (40, 2, 64, 16, [(0, 9), (70, 20)]),   # a group of 20
])
def test_prefill(h, hkv, d, bs, spans, dtype, fmt):
    if dtype != torch.float32:
        check_prefill(h, hkv, d, bs, spans, dtype, fmt, 2)
        return
    rows = sum(n for _, n in spans)
    few = rows * max(7 * hkv, h) <= 2240 and h // hkv <= 16
    check_prefill(h, hkv, d, bs, spans, dtype, fmt, 1 if few else 4)
    check_prefill(h, hkv, d, bs, spans, dtype, fmt, 4, more=2300)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs,width", [(16, 0), (16, 4000), (12, 0), (1, 7), (256, 0)])
def test_prefill_layouts(bs, width, dtype):
    """Dense and in-place expansion (a wide table), blocks of any size, and
    nothing read that no row attends."""
    check_prefill(8, 2, 64, bs, [(0, 70), (33, 2), (0, 1), (260, 140)], dtype, "e4m3",
                  2 if dtype == torch.bfloat16 else 4, width=width, dirty=True)
    more = 2300 if dtype == torch.float32 else 0
    check_prefill(8, 2, 64, bs, [(0, 70), (33, 20)], dtype, "int8",
                  2 if dtype == torch.bfloat16 else 4, width=width, more=more)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prefill_few_rows_and_forced_paths(dtype):
    spans = [(100, 1), (0, 1), (33, 4), (500, 2)]
    check_prefill(28, 4, 128, 16, spans, dtype, "e4m3", 1)
    if dtype == torch.bfloat16:
        ops.set_prefill_path(2)
        try:
            check_prefill(28, 4, 128, 16, spans, dtype, "e4m3", 2)
        finally:
            ops.set_prefill_path(0)
    ops.set_prefill_path(1)
    try:
        check_prefill(28, 4, 128, 16, spans, dtype, "e4m3", 1)
        check_prefill(28, 4, 128, 16, [(3, 70), (10, 9)], dtype, "int8", 4, spread=4.0,
                      more=2300)
    finally:
        ops.set_prefill_path(0)


@pytest.mark.parametrize("dtype,fmt", [(torch.bfloat16, "e4m3"), (torch.float16, "int8")])
def test_prefill_mixed_frame(dtype, fmt):
    """Wide tables and both long and short sequences: those of up to 8 rows are
    decoded from the codes, the others expanded; rows of neither stay."""
    spans = [(300, 1), (0, 200), (500, 8), (100, 9), (20, 0), (64, 1)]
    for bs in (16, 32):
        check_prefill(28, 4, 128, bs, spans, dtype, fmt, 2, width=400, dirty=True)
    check_prefill(8, 1, 64, 8, spans, dtype, fmt, 2, width=800, dirty=True)
    f = wl.prefill_frame("t", 3, [s for s, _ in spans], [n for _, n in spans], 8, 2, 64, 16)
    kc, ks = make_pool(np.random.default_rng(1), f.num_blocks, 16, 2, 64, fmt)
    pool, sc = codes_to(kc, fmt), dev(ks.astype(np.float32))
    q = dev(np.random.default_rng(2).normal(size=(250, 8, 64))).to(dtype)
    out = torch.full_like(q, 7.0)
    call = lambda q, **kw: irb.paged_prefill_q8(  # noqa: E731
        q, pool, pool, sc, sc, dev(np.pad(f.block_tables, ((0, 0), (0, 400)))),
        dev(f.context_lens), dev(f.q_start), f.scale, 16, **kw)
    call(q, out=out)
    assert (out[219:] == 7.0).all() and torch.equal(out[:219], call(q[:219]))
    bad = f.context_lens.copy()
    bad[0] = 0                                    # a short sequence, then a long one
    bad[1] = 100
    irb.paged_prefill_q8(q, pool, pool, sc, sc, dev(np.pad(f.block_tables, ((0, 0), (0, 400)))),
                         dev(bad), dev(f.q_start), f.scale, 16, out=out.fill_(7.0))
    with pytest.raises(irb.DeviceError, match="CONTEXT_LEN"):
        irb.check_device_errors()
    good = call(q[:219])
    assert torch.equal(out[209:218], good[209:218])
    # decoded rows are cut into pieces by the lengths of all of them: each result
    # is within one output rounding (at most 2^-8), one of the weights (2^-11) and
    # the scores' (72 * 2^-23 * 100 < 2^-10) of the same weighted mean of V
    top = np.abs(q8.values(kc, ks, 16)).max()
    rest = [*range(201, 209), 218]
    assert (np.abs(host(out[rest]) - host(good[rest])) <= 2 * (2.0 ** -8 + 2.0 ** -9) * top).all()


def test_prefill_unaligned_rows():
    rng = np.random.default_rng(4)
    n, h, d = 29, 8, 64
    for off, stride, path in ((1, h * d + 3, 4), (1, h * d + 8, 2), (0, h * d + 64, 2)):
        flat = dev(rng.normal(size=n * (h * d + 64) + 16)).to(torch.bfloat16)
        q = flat[off:].as_strided((n, h, d), (stride, d, 1), off)
        check_prefill(h, 2, d, 16, [(20, 20), (0, 9)], torch.bfloat16, "e4m3", path, q=q)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prefill_nan_reaches_the_rows_that_attend_it(dtype, fmt):
    """A NaN in K or V at one position: rows before it keep their values, to the bit."""
    rng = np.random.default_rng(2)
    h, hkv, d, bs, n = 8, 2, 64, 16, 90
    f = wl.prefill_frame("t", 3, [10, 0], [n, 30], h, hkv, d, bs)
    kc, ks = make_pool(rng, f.num_blocks, bs, hkv, d, fmt)
    vc, vs = make_pool(rng, f.num_blocks, bs, hkv, d, fmt)
    q = dev(rng.normal(size=(f.total_q, h, d))).to(dtype)
    bt, ctx, qs = dev(f.block_tables), dev(f.context_lens), dev(f.q_start)

    def run(kc, ks, vc, vs):
        return irb.paged_prefill_q8(q, codes_to(kc, fmt), codes_to(vc, fmt),
                                    dev(ks.astype(np.float32)), dev(vs.astype(np.float32)), bt,
                                    ctx, qs, f.scale, bs)

    clean = run(kc, ks, vc, vs)
    at = 64   # a block's first position, so that an int8 scale begins there
    slot = f.block_tables[0, at // bs] * bs + at % bs
    for side in "vk":
        k2, v2, ks2, vs2 = kc.copy(), vc.copy(), ks.copy(), vs.copy()
        if fmt == "e4m3":
            (v2 if side == "v" else k2)[slot, 1, 5] = np.nan
        else:
            (vs2 if side == "v" else ks2)[slot // bs, 1] = np.nan
        out = run(k2, ks2, v2, vs2)
        bad = torch.isnan(out)
        want = torch.zeros_like(bad)
        rows = slice(at - 10, n)
        if side == "v" and fmt == "e4m3" and dtype == torch.float32:
            want[rows, 4:, 5] = True
        else:   # (the tensor-core path: the whole head)
            want[rows, 4:] = True
        assert torch.equal(bad, want)
        assert torch.equal(out[~want], clean[~want])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prefill_bad_metadata_is_flagged(dtype):
    rng = np.random.default_rng(2)
    f = wl.prefill_frame("t", 3, [10, 0], [40, 30], 8, 2, 64, 16)
    kc, ks = make_pool(rng, f.num_blocks, 16, 2, 64, "e4m3")
    pool, sc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32))
    q = dev(rng.normal(size=(70, 8, 64))).to(dtype)
    run = lambda bt, ctx: irb.paged_prefill_q8(q, pool, pool, sc, sc, dev(bt), dev(ctx),  # noqa: E731
                                               dev(f.q_start), f.scale, 16)
    good = run(f.block_tables, f.context_lens)
    bt = f.block_tables.copy()
    bt[0, 1] = f.num_blocks
    out = run(bt, f.context_lens)
    with pytest.raises(irb.DeviceError, match="BLOCK_ID"):
        irb.check_device_errors()
    assert torch.equal(out[40:], good[40:])
    for c in (np.array([30, 30], np.int32), np.array([16 * 4 + 1, 30], np.int32)):
        out = run(f.block_tables, c)
        with pytest.raises(irb.DeviceError, match="CONTEXT_LEN"):
            irb.check_device_errors()
        assert torch.equal(out[40:], good[40:])
    # rows behind the last sequence stay as they were
    out = torch.full_like(q, 7.0)
    irb.paged_prefill_q8(q, pool, pool, sc, sc, dev(f.block_tables[:1]), dev(f.context_lens[:1]),
                         dev(f.q_start[:2]), f.scale, 16, out=out)
    assert (out[40:] == 7.0).all() and torch.equal(out[:40], good[:40])


@pytest.mark.parametrize("path,dtype", [(2, torch.bfloat16), (1, torch.bfloat16),
                                        (1, torch.float32)])
def test_prefill_few_rows_leave_the_others_alone(path, dtype):
    """One or two rows per sequence, with rows of no sequence behind them."""
    rng = np.random.default_rng(5)
    f = wl.prefill_frame("t", 3, [10, 0, 300], [1, 2, 1], 8, 2, 64, 16)
    kc, ks = make_pool(rng, f.num_blocks, 16, 2, 64, "e4m3")
    pool, sc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32))
    q = dev(rng.normal(size=(9, 8, 64))).to(dtype)
    args = (pool, pool, sc, sc, dev(f.block_tables), dev(f.context_lens), dev(f.q_start), f.scale,
            16)
    ops.set_prefill_path(2 if path == 2 else 0)
    try:
        assert ops.prefill_plan_q8(q, pool, args[4], args[6], 16)[0] == path
        good = irb.paged_prefill_q8(q[:4], *args)
        out = torch.full_like(q, 7.0)
        irb.paged_prefill_q8(q, *args, out=out)
    finally:
        ops.set_prefill_path(0)
    assert torch.equal(out[:4], good) and (out[4:] == 7.0).all()


def test_prefill_overflow_of_later_positions_stays_there():
    """A V whose code times its scale is beyond the type is held as its largest
    value: rows before it do not meet an infinity."""
    rng = np.random.default_rng(6)
    f = wl.prefill_frame("t", 3, [0], [60], 4, 2, 64, 16)
    kc, ks = make_pool(rng, f.num_blocks, 16, 2, 64, "e4m3")
    q = dev(rng.normal(size=(60, 4, 64))).to(torch.bfloat16)
    run = lambda c, s: irb.paged_prefill_q8(  # noqa: E731
        q, codes_to(kc, "e4m3"), codes_to(c, "e4m3"), dev(ks.astype(np.float32)),
        dev(s.astype(np.float32)), dev(f.block_tables), dev(f.context_lens), dev(f.q_start),
        f.scale, 16)
    clean = run(kc, ks)
    vc, vs = kc.copy(), ks.copy()
    blk = int(f.block_tables[0, 2])            # positions 32 .. 47
    vc[blk * 16:(blk + 1) * 16] = 448.0
    vs[blk] = 2.0 ** 120
    assert torch.equal(run(vc, vs)[:32], clean[:32])


def test_prefill_row_is_the_decode_row():
    """A prompt's last row and the decode of the same token agree within both bounds."""
    rng = np.random.default_rng(0)
    h, hkv, d, bs = 28, 4, 128, 16
    f = wl.prefill_frame("t", 3, [0], [100], h, hkv, d, bs)
    kc, ks = make_pool(rng, f.num_blocks, bs, hkv, d, "e4m3")
    q = dev(rng.normal(size=(100, h, d))).to(torch.bfloat16)
    pool, sc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32))
    bt, ctx = dev(f.block_tables), dev(f.context_lens)
    a = irb.paged_prefill_q8(q, pool, pool, sc, sc, bt, ctx, dev(f.q_start), f.scale, bs)[-1]
    b = irb.paged_decode_q8(q[-1:], pool, pool, sc, sc, bt, ctx, f.scale, bs)[0]
    _, weighted, _ = q8.attend(host(q[99]), *[q8.history(q8.values(kc, ks, bs), f.block_tables[0],
                                                         100, bs)] * 2, f.scale)
    # two output roundings and P in bf16 (2^-8) and fp16 (2^-11)
    assert (np.abs(host(a) - host(b)) <= (2 * 2.0 ** -8 + 2 * 2.0 ** -8 + 2.0 ** -10) * weighted).all()


# ---------------------------------------------------------------- a run of them together


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_prompt_then_decode_steps(fmt):
    """norm + rotation, quantising write, prefill and decode as one layer of a
    model would run them, each step against 64 bits on the same codes."""
    rng = np.random.default_rng(11)
    h, hkv, d, bs, nb = 14, 2, 64, 16, 12
    dt = torch.bfloat16
    kp, vp = (torch.zeros(nb * bs, hkv, d, dtype=torch.int8, device=DEV).view(FMT[fmt])
              for _ in range(2))
    ks, vs = (torch.zeros(nb, hkv, device=DEV) for _ in range(2))
    table = rng.permutation(nb).astype(np.int32)[None]
    wq, wk = (dev(1 + 0.1 * rng.normal(size=d)).to(dt) for _ in range(2))
    inv = 1e4 ** (-np.arange(0, d, 2) / d)
    pos = 0
    for n in (37, 1, 1, 9, 1):
        x = dev(rng.normal(size=(n, (h + 2 * hkv) * d))).to(dt)
        p = np.arange(pos, pos + n)
        ang = np.concatenate([p[:, None] * inv] * 2, axis=1)
        cos, sin = dev(np.cos(ang).astype(np.float32)), dev(np.sin(ang).astype(np.float32))
        q, k = irb.qk_norm_rope(x[:, :h * d].view(n, h, d),
                                x[:, h * d:(h + hkv) * d].view(n, hkv, d), wq, wk, cos, sin, 1e-6)
        slots = table[0, p // bs].astype(np.int64) * bs + p % bs
        irb.cache_write_q8(k, x[:, (h + hkv) * d:].view(n, hkv, d), kp, vp, ks, vs, dev(slots), bs)
        pos += n
        ctx = dev(np.array([pos], np.int32))
        if n == 1:
            out = irb.paged_decode_q8(q, kp, vp, ks, vs, dev(table), ctx, d ** -0.5, bs)
        else:
            out = irb.paged_prefill_q8(q, kp, vp, ks, vs, dev(table), ctx,
                                       dev(np.array([0, n], np.int32)), d ** -0.5, bs)
        kv, vv = (q8.values(host(c), host(s), bs) for c, s in ((kp, ks), (vp, vs)))
        for r in range(n):
            t = pos - n + r + 1
            want, weighted, size = q8.attend(host(q[r]), q8.history(kv, table[0], t, bs),
                                             q8.history(vv, table[0], t, bs), d ** -0.5)
            tol = attend_tolerance(want, weighted, size, t, d, dt, False) + 2 * 2.0 ** -8 * weighted
            assert (np.abs(host(out[r]) - want) <= tol).all()
    # what the cache holds is off by the quantisation alone
    back = irb.cache_gather_q8(kp, ks, dev(slots), bs, torch.float32)
    unit = ks.max().item() * (0.5 if fmt == "int8" else 16)
    assert (back - k.float()).abs().max().item() <= 2 * unit


# ---------------------------------------------------------------- pool, seam, streams, graphs


def test_pool_scales_are_fp32_under_another_default_type():
    torch.set_default_dtype(torch.bfloat16)
    try:
        pool = irb.PagedKVPoolQ8(1, 2, 16, 1, 64, torch.bfloat16)
    finally:
        torch.set_default_dtype(torch.float32)
    assert pool.k_scale.dtype == pool.v_scale.dtype == torch.float32


@pytest.mark.parametrize("kv", [torch.float8_e4m3fn, torch.int8])
def test_pool_class_and_paged_attention(kv):
    """``paged_attention`` on a two-layer 8-bit pool: a packed frame, then a decode
    step, as the direct calls on the same codes give them."""
    from oracle import paged_attention_np as orc

    rng = np.random.default_rng(4)
    h, hkv, d, bs, nb = 14, 2, 64, 16, 20
    dt = torch.bfloat16
    pool = irb.PagedKVPoolQ8(2, nb, bs, hkv, d, dt, kv)
    assert pool.k.dtype == kv and pool.num_slots == nb * bs
    starts, qls = [0, 0], [20, 37]
    bt = rng.permutation(nb)[:8].reshape(2, 4).astype(np.int32)
    fr = orc.varlen_frame(bt, starts, qls, bs)
    n = sum(qls)
    q = dev(rng.normal(size=(1, n, h, d))).to(dt)
    k, v = (dev(rng.normal(size=(1, n, hkv, d))).to(dt) for _ in range(2))
    gs = dev(fr["gather_slots"]).reshape(1, -1)
    ws = dev(fr["write_slots"])
    mask = dev(orc.varlen_mask(fr["q_seq_ids"], fr["q_pos"], fr["k_seq_ids"], fr["k_pos"]))
    paged = irb.PagedContext(pool, ws, gs)
    out = irb.paged_attention(q, k, v, paged, mask, 1, d ** -0.5, h // hkv)
    q_start = dev(np.array([0, 20, 57], np.int32))
    ctx = dev(np.array(qls, np.int32))
    want = irb.paged_prefill_q8(q[0], *pool.layer(1), dev(bt), ctx, q_start, d ** -0.5, bs)
    assert torch.equal(out[0], want)
    back = pool.gather(1, gs)
    assert back[0].shape == (1, n, hkv, d) and back[0].dtype == dt
    assert not pool.k[0].view(torch.int8).any()   # the other layer is untouched
    # each row is off by its quantisation alone: half a code unit
    kf = k[0].float()
    unit = 2.0 ** -4 * kf.abs() + 2.0 ** -10 * pool.k_scale[1].max() if kv != torch.int8 else \
        pool.k_scale[1].max() / 2
    rows = irb.cache_gather_q8(pool.k[1], pool.k_scale[1], ws, bs, torch.float32)
    assert ((rows - kf).abs() <= unit).all()
    # a decode step for both sequences
    ctx1 = np.array(qls, np.int32) + 1
    t = int(ctx1.max())
    gs1 = dev(orc.gather_slots_from_tables(bt, ctx1, bs, t))
    m1 = dev(orc.decode_mask(ctx1, t))
    ws1 = dev(wl.tail_slots(bt, ctx1, bs))
    q1 = dev(rng.normal(size=(2, 1, h, d))).to(dt)
    k1, v1 = (dev(rng.normal(size=(2, 1, hkv, d))).to(dt) for _ in range(2))
    got = irb.paged_attention(q1, k1, v1, irb.PagedContext(pool, ws1, gs1), m1, 1, d ** -0.5,
                              h // hkv)
    want = irb.paged_decode_q8(q1[:, 0], *pool.layer(1), dev(bt), dev(ctx1), d ** -0.5, bs)
    assert torch.equal(got[:, 0], want)


def test_pool_class_refusals():
    with pytest.raises(ValueError):
        irb.PagedKVPoolQ8(1, 2, 16, 2, 64, torch.bfloat16, device="cpu")
    with pytest.raises(irb.UnsupportedShape):
        irb.PagedKVPoolQ8(1, 2, 16, 2, 64, torch.bfloat16, torch.uint8)
    with pytest.raises(irb.UnsupportedShape):
        irb.PagedKVPoolQ8(1, 2, 16, 2, 64, torch.float64)


def test_python_refusals():
    rng = np.random.default_rng(0)
    codes, scale = make_pool(rng, 4, 16, 2, 64, "e4m3")
    p, sc = codes_to(codes, "e4m3"), dev(scale.astype(np.float32))
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=DEV)
    slots = dev(np.arange(3))
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    bt, ctx = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    qs = dev(np.array([0, 1, 2], np.int32))
    write = lambda **o: irb.cache_write_q8(*{**dict(k=k, v=k, kp=p, vp=p, ks=sc, vs=sc, s=slots,  # noqa: E731
                                                    bs=16), **o}.values())
    decode = lambda **o: irb.paged_decode_q8(*{**dict(q=q, kp=p, vp=p, ks=sc, vs=sc, bt=bt, c=ctx,  # noqa: E731
                                                      f=0.1, bs=16), **o}.values())
    for bad in (dict(ks=sc.double()), dict(ks=sc[:2]), dict(vs=sc.t().contiguous()), dict(bs=12),
                dict(bs=0), dict(vp=codes_to(codes, "int8")), dict(kp=p[:, :1]), dict(vp=p[:48])):
        with pytest.raises((ValueError, irb.InfraredB200Error)):
            write(**bad)
        with pytest.raises((ValueError, irb.InfraredB200Error)):
            decode(**bad)
    for bad in (dict(k=k.half()), dict(s=slots.int()), dict(s=dev(np.arange(4))), dict(k=k.double()),
                dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)), dict(s=slots.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            write(**bad)
    for bad in (dict(q=q[:1]), dict(q=q[0]), dict(bt=bt.long()), dict(c=ctx[:1]), dict(q=q.double()),
                dict(q=torch.zeros(2, 3, 64, dtype=q.dtype, device=DEV)), dict(bt=bt.cpu())):
        with pytest.raises((ValueError, irb.InfraredB200Error)):
            decode(**bad)
    with pytest.raises(ValueError):
        irb.paged_decode_q8(q, p, p, sc, sc, bt, ctx, 0.1, 16, out=torch.empty(2, 4, 65, device=DEV))
    with pytest.raises(ValueError):
        irb.paged_decode_q8(q, p, p, sc, sc, bt, ctx, 0.1, 16,
                            ws=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        irb.paged_prefill_q8(q, p, p, sc, sc, bt, ctx, qs[:2], 0.1, 16)
    with pytest.raises(ValueError):
        irb.cache_gather_q8(p, sc, slots.int(), 16, torch.float32)


def test_kernel_choice_can_change_between_equal_calls():
    """The same call with the CUDA-core kernel asked for in between."""
    w = _with_lengths(5, [600, 33, 1], 14, 2, 64, 16)
    a = check_decode(w, "e4m3", torch.bfloat16, 2)
    ops.set_decode_path(1)
    try:
        b = check_decode(w, "e4m3", torch.bfloat16, 1)
    finally:
        ops.set_decode_path(0)
    c = check_decode(w, "e4m3", torch.bfloat16, 2)
    assert torch.equal(a, c) and a.shape == b.shape


@pytest.mark.parametrize("n", [9, 1500])
def test_write_and_gather_on_a_side_stream_and_in_a_graph(n):
    rng = np.random.default_rng(n)
    codes, scale, rows, slots = _write_case(rng, n, 2, 64, 16, 100, "e4m3", torch.bfloat16)
    want, ws = codes.copy(), scale.copy()
    q8.write(want, ws, host(rows[0]), slots, 16, "e4m3")
    s = dev(slots.astype(np.int64))

    def fresh():
        return (codes_to(codes, "e4m3"), codes_to(codes, "e4m3"),
                dev(scale.astype(np.float32)), dev(scale.astype(np.float32)))

    side = torch.cuda.Stream()
    kp, vp, ks, vs = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        irb.cache_write_q8(rows[0], rows[1], kp, vp, ks, vs, s, 16)
        got = irb.cache_gather_q8(kp, ks, s, 16, torch.float32)
    side.synchronize()
    np.testing.assert_array_equal(host(kp), want)
    np.testing.assert_array_equal(host(got), q8.values(want, ws, 16)[slots])
    # captured, with other rows replayed through the same buffers
    kp, vp, ks, vs = fresh()
    k2, v2 = torch.zeros_like(rows[0]), torch.zeros_like(rows[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        irb.cache_write_q8(k2, v2, kp, vp, ks, vs, s, 16)
        got = irb.cache_gather_q8(kp, ks, s, 16, torch.float32)
    kp.view(torch.int8).copy_(fresh()[0].view(torch.int8))
    ks.copy_(fresh()[2])
    for rep in range(2):   # the second replay finds the scales grown and changes nothing
        k2.copy_(rows[0])
        v2.copy_(rows[1])
        g.replay()
        torch.cuda.synchronize()
        if rep == 0:
            np.testing.assert_array_equal(host(kp), want)
            np.testing.assert_array_equal(host(ks), ws)
        np.testing.assert_array_equal(host(got), q8.values(want, ws, 16)[slots])


def test_a_long_table_passes_32_bits_of_bytes():
    """Codes beyond 2^31 bytes into the pool, and rows of the expanded pool beyond it."""
    hkv, d, bs = 8, 128, 16
    nb = (2 ** 31 // (hkv * d)) // bs + 40   # the last blocks lie past 2^31 bytes
    kp = torch.zeros(nb * bs, hkv, d, dtype=torch.int8, device=DEV).view(torch.float8_e4m3fn)
    vp = torch.zeros_like(kp.view(torch.int8)).view(torch.float8_e4m3fn)
    ks, vs = torch.zeros(nb, hkv, device=DEV), torch.zeros(nb, hkv, device=DEV)
    rng = np.random.default_rng(1)
    n = 100
    bt = np.array([[nb - 1, nb - 9, nb - 4, 3, nb - 2, nb - 30, nb - 7]], np.int32)
    p = np.arange(n)
    slots = bt[0, p // bs].astype(np.int64) * bs + p % bs
    k, v = (dev(rng.normal(size=(n, hkv, d))).to(torch.bfloat16) for _ in range(2))
    irb.cache_write_q8(k, v, kp, vp, ks, vs, dev(slots), bs)
    kf = irb.cache_gather_q8(kp, ks, dev(slots), bs, torch.float32)
    vf = irb.cache_gather_q8(vp, vs, dev(slots), bs, torch.float32)
    assert ((kf - k.float()).abs() <= 2.0 ** -4 * k.float().abs() + 2.0 ** -10 * ks.max()).all()
    q = dev(rng.normal(size=(1, 16, d))).to(torch.bfloat16)
    ctx = dev(np.array([n], np.int32))
    out = irb.paged_decode_q8(q, kp, vp, ks, vs, dev(bt), ctx, d ** -0.5, bs)
    want, weighted, size = q8.attend(host(q[0]), host(kf), host(vf), d ** -0.5)
    assert (np.abs(host(out[0]) - want) <=
            attend_tolerance(want, weighted, size, n, d, torch.bfloat16, True)).all()


# ---------------------------------------------------------------- contexts past the table


@pytest.mark.parametrize("over", [1, 63, 64])
@pytest.mark.parametrize("dtype,d,force", [
    (torch.bfloat16, 64, 0), (torch.float16, 64, 0), (torch.float32, 64, 0),
    (torch.bfloat16, 128, 2), (torch.bfloat16, 128, 3), (torch.bfloat16, 64, 1)])
def test_prefill_context_past_the_table_leaves_its_rows_alone(dtype, d, force, over):
    """A context that the table does not hold is flagged and its rows stay as they
    were, on every path: nothing that the call's workspace held before comes out."""
    rng = np.random.default_rng(2)
    f = wl.prefill_frame("t", 3, [10, 0], [40, 30], 8, 2, d, 16)
    kc, ks = make_pool(rng, f.num_blocks, 16, 2, d, "e4m3")
    pool, sc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32))
    q = dev(rng.normal(size=(70, 8, d))).to(dtype)
    bt, qs = dev(f.block_tables), dev(f.q_start)
    held = 16 * f.block_tables.shape[1]
    ops.set_prefill_path(force)
    try:
        _, nbytes = ops.prefill_plan_q8(q, pool, bt, qs, 16)
        for first in (held + over, held):
            ws = torch.full((max(nbytes, 256),), 0xff, dtype=torch.uint8, device=DEV)
            out = torch.full_like(q, 7.0)
            irb.paged_prefill_q8(q, pool, pool, sc, sc, bt, dev(np.array([first, 30], np.int32)),
                                 qs, f.scale, 16, out=out, ws=ws)
            if first > held:
                with pytest.raises(irb.DeviceError, match="CONTEXT_LEN"):
                    irb.check_device_errors()
                assert (out[:40] == 7.0).all()
                rest = out[40:].clone()
    finally:
        ops.set_prefill_path(0)
    assert not (out[:40] == 7.0).all() and torch.isfinite(out).all()
    if force != 1:   # (rows decoded one by one are cut by the lengths of all)
        assert torch.equal(out[40:], rest)


# ---------------------------------------------------------------- fp16 rows, values beyond fp16


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("side", ["large k", "large v", "small k", "both"])
@pytest.mark.parametrize("d,bs,width,force", [(64, 16, 0, 0), (128, 16, 4000, 0), (64, 12, 0, 0),
                                              (128, 16, 0, 3)])
def test_prefill_fp16_over_values_beyond_its_range(d, bs, width, force, side, fmt):
    """A pool written from wider rows holds values that fp16 does not: the rows that
    attend one are held to the fp32 kernel's bound (no rounding of weights or of
    the history), those before keep their bits, as do other sequences; codes past
    the context decide nothing."""
    rng = np.random.default_rng(6)
    h, hkv, n, head = 8, 2, 150, 31
    f = wl.prefill_frame("t", 3, [head, 0, 5], [n, 20, 70], h, hkv, d, bs)
    kc, ks0 = make_pool(rng, f.num_blocks, bs, hkv, d, fmt)
    vc, vs0 = make_pool(rng, f.num_blocks, bs, hkv, d, fmt)
    table = f.block_tables[0, :-(-(head + n) // bs)]
    # the last block: small codes and then, past the context, one that fp16 cannot hold
    past = (head + n) % bs
    at = table[-1] * bs
    vc[at:at + bs] = np.sign(vc[at:at + bs])
    vs0[table[-1]] = 2.0 ** (8 if fmt == "e4m3" else 10)
    vx = vc.copy()
    vx[at + past:at + bs] = 448 if fmt == "e4m3" else 127
    ks, vs, scale, qsize = ks0.copy(), vs0.copy(), f.scale, 1.0
    blk = table[70 // bs]
    if side in ("large v", "both"):        # up to 114688 or 130048
        vs[blk] = 2.0 ** (8 if fmt == "e4m3" else 10)
    if side in ("large k", "both"):
        ks[blk, 1] = 2.0 ** (10 if fmt == "e4m3" else 12)
        qsize = 2.0 ** -16
    if side == "small k":                  # scores of usual size from large q and scale
        ks[table] *= 2.0 ** -22 if fmt == "e4m3" else 2.0 ** -24
        scale, qsize = scale * 2.0 ** 12, 2.0 ** 10
    q = dev(rng.normal(size=(f.total_q, h, d)) * qsize).to(torch.float16)
    bt = dev(np.pad(f.block_tables, ((0, 0), (0, width))))

    def run(ks, vs, vc=vc):
        return irb.paged_prefill_q8(q, codes_to(kc, fmt), codes_to(vc, fmt),
                                    dev(ks.astype(np.float32)), dev(vs.astype(np.float32)), bt,
                                    dev(f.context_lens), dev(f.q_start), scale, bs)

    ops.set_prefill_path(force)
    try:
        assert ops.prefill_plan_q8(q, codes_to(kc, fmt), bt, dev(f.q_start), bs)[0] == (force or 2)
        got, clean = run(ks, vs), run(ks0, vs0)
        assert torch.equal(run(ks0, vs0, vx), clean)
    finally:
        ops.set_prefill_path(0)
    kh = q8.history(q8.values(kc, ks, bs), f.block_tables[0], head + n, bs)
    vh = q8.history(q8.values(vc, vs, bs), f.block_tables[0], head + n, bs)
    lost = (np.abs(kh) > 65504) | (np.abs(vh) > 65504) | \
        ((np.abs(kh) < 2.0 ** -14) & (np.clip(kh, -1, 1).astype(np.float16) != kh))
    start = int(np.nonzero(lost.any(axis=(1, 2)))[0][0])
    assert side == "small k" or 70 // bs * bs <= start < (70 // bs + 1) * bs
    before = max(start - head, 0)          # rows of the first sequence that attend none of them
    same = 0 if side == "small k" else 70 // bs * bs - head   # nor another row of their block
    assert torch.equal(got[:same], clean[:same]) and torch.equal(got[n:], clean[n:])
    g, qh = host(got), host(q)
    for r in (*range(same, before), *range(before, n, 3)):
        t = head + r + 1
        want, weighted, size = q8.attend(qh[r], kh[:t], vh[:t], scale)
        tol = attend_tolerance(want, weighted, size, t, d, torch.float16, False)
        if r < before:                     # the tensor cores' rows, as in check_prefill
            tol = tol + 2.0 ** -10 * weighted + t * 2.0 ** -25 * np.abs(vh[:t]).max() + 2.0 ** -24
        # (an output that rounds beyond fp16 is infinite: 65520 is half way to 2^16)
        over = np.abs(want) - tol > 65520
        assert (g[r][over] == np.sign(want[over]) * np.inf).all()
        sure = np.abs(want) + tol < 65520
        assert (np.abs(g[r] - want)[sure] <= tol[sure]).all(), r


# ---------------------------------------------------------------- blocks whose scale grows


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("seqs,hkv,d,bs", [(3, 2, 64, 16), (5, 1, 128, 32), (1100, 1, 64, 16),
                                           (1030, 2, 64, 8)])
def test_write_growing_blocks_stay_near_their_rows(seqs, hkv, d, bs, fmt):
    """Blocks filled token by token (one call a step, on the short and the long path)
    by rows that grow, so that most steps raise the scale: what is read back
    against the rows themselves. A value goes through scales of which each is at
    most half of the next: int8 is off by half a unit of each, less than one unit
    of the last; e4m3 by 2^-4 of the value, and where it is subnormal by half of
    2^-9 of each scale, less than 2^-9 of the last."""
    rng = np.random.default_rng(bs + seqs)
    size = 2.0 ** (rng.uniform(0.3, 1.0, size=(seqs, bs, 1, 1)).cumsum(axis=1) - 6)
    x = dev(rng.normal(size=(seqs, bs, hkv, d)) * size).to(torch.bfloat16)
    pools = [torch.zeros(seqs * bs, hkv, d, dtype=torch.int8, device=DEV).view(FMT[fmt])
             for _ in range(2)]
    scales = [torch.zeros(seqs, hkv, device=DEV) for _ in range(2)]
    table = dev(rng.permutation(seqs))
    raised = 0
    for i in range(bs):
        before = scales[0].clone()
        row = x[:, i].contiguous()
        irb.cache_write_q8(row, -row, *pools, *scales, table * bs + i, bs)
        raised += int((scales[0] > before).sum())
    assert raised > seqs * hkv * bs // 3
    slots = (table[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)
    want = x.reshape(seqs * bs, hkv, d).double()
    for pool, scale, sign in zip(pools, scales, (1, -1)):
        back = irb.cache_gather_q8(pool, scale, slots, bs, torch.float32).double() * sign
        last = scale[table].double().repeat_interleave(bs, dim=0)[..., None]
        tol = last if fmt == "int8" else 2.0 ** -4 * want.abs() + 2.0 ** -9 * last
        assert ((back - want).abs() < tol).all()


def test_write_one_block_of_two_runs_in_a_long_call():
    """A long call in order but for one block, whose rows come in two runs."""
    rng = np.random.default_rng(3)
    n, bs, nb = 3000, 16, 200
    for fmt in ("e4m3", "int8"):
        codes, scale, rows, slots = _write_case(rng, n, 2, 64, bs, nb, fmt, torch.bfloat16, "runs")
        at = np.nonzero(slots // bs == slots[1500] // bs)[0]   # one row of it to the front
        order = np.concatenate([at[1:2], np.delete(np.arange(n), at[1])])
        _check_write(codes, scale, [x[dev(order)] for x in rows], slots[order], bs, fmt)


# ---------------------------------------------------------------- frames of a serving step


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("chunk,path", [(150, 1), (400, 2)])
def test_prefill_many_single_rows_and_a_chunk(chunk, path, dtype):
    """A step of many decode rows and a chunk of a prompt: with few rows on average
    all are decoded, the chunk's too; else the single rows are, beside it."""
    spans = [(7 * i, 1) for i in range(25)] + [(130, chunk)] + [(50, 1)] * 5
    check_prefill(14, 2, 64, 16, spans, dtype, "e4m3", path, width=60)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prefill_many_sequences_under_a_wide_table(dtype):
    """Tables far wider than any context (as a packed frame's seam makes them), where
    the history is expanded in the blocks' own places."""
    spans = [(5 * i, 1) for i in range(30)] + [(40, 333)]
    check_prefill(8, 2, 64, 16, spans, dtype, "int8", 4 if dtype == torch.float32 else 2,
                  width=9400, dirty=True)
    check_prefill(8, 2, 64, 16, spans[:30], dtype, "e4m3", 1, width=9400)


# ---------------------------------------------------------------- rows outside the frame


@pytest.mark.parametrize("pool8", [True, False])
@pytest.mark.parametrize("dtype,force", [(torch.bfloat16, 2), (torch.float16, 2), (torch.bfloat16, 3),
                                         (torch.float32, 0), (torch.bfloat16, 1)])
@pytest.mark.parametrize("q_start", [[0, 40, 300], [-60, 40, 70], [0, 40, 2 ** 31 - 1],
                                     [-2 ** 31, 40, 70]])
def test_prefill_rows_outside_the_frame_write_nothing(q_start, dtype, force, pool8):
    """q_start that reaches past the packed rows, or before them: the sequence's rows
    outside are not written (here they lie in the same buffer, before and behind)."""
    rng = np.random.default_rng(2)
    n, h, hkv, d, bs = 70, 8, 2, 128, 16
    f = wl.prefill_frame("t", 3, [300, 300], [40, 30], h, hkv, d, bs)
    kc, ks = make_pool(rng, f.num_blocks, bs, hkv, d, "e4m3")
    pool, sc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32))
    rows = dev(q8.values(kc, ks, bs).astype(np.float32)).to(dtype)
    q = dev(rng.normal(size=(n, h, d))).to(dtype)
    bt, ctx = dev(f.block_tables), dev(f.context_lens)
    good = q_start[0] == 0   # the first sequence is sound, else the second

    def run(start):
        room = torch.full((512 + n + 512, h, d), 7.0, dtype=dtype, device=DEV)
        out = room[512:512 + n]
        starts = dev(np.array(start, np.int32))
        if pool8:
            irb.paged_prefill_q8(q, pool, pool, sc, sc, bt, ctx, starts, f.scale, bs, out=out)
        else:
            irb.paged_prefill(q, rows, rows, bt, ctx, starts, f.scale, bs, out=out)
        return room, out

    ops.set_prefill_path(force)
    try:
        _, want = run([0, 40, 70])
        room, out = run(q_start)
    finally:
        ops.set_prefill_path(0)
    torch.cuda.synchronize()
    ops.error_flag().zero_()   # (the tensor-core and tile kernels flag it, decoded rows do not)
    assert (room[:512] == 7.0).all() and (room[512 + n:] == 7.0).all()
    if force >= 2:
        assert torch.equal(out[:40] if good else out[40:], want[:40] if good else want[40:])
        assert (out[40:] == 7.0).all() if good else (out[:40] == 7.0).all()


def test_prefill_fp16_graph_follows_the_scales():
    """A captured fp16 prefill whose pool's scales change between replays: which rows
    leave the tensor cores is found anew each time, on another stream too."""
    rng = np.random.default_rng(8)
    f = wl.prefill_frame("t", 3, [40, 0], [100, 60], 8, 2, 64, 16)
    kc, ks = make_pool(rng, f.num_blocks, 16, 2, 64, "e4m3")
    pool, sc, vsc = codes_to(kc, "e4m3"), dev(ks.astype(np.float32)), dev(ks.astype(np.float32))
    q = dev(rng.normal(size=(160, 8, 64))).to(torch.float16)
    bt, ctx, qs = dev(f.block_tables), dev(f.context_lens), dev(f.q_start)
    call = lambda **kw: irb.paged_prefill_q8(q, pool, pool, sc, vsc, bt, ctx, qs, f.scale, 16,  # noqa: E731
                                             **kw)
    large = vsc.clone()
    large[int(f.block_tables[0, 4])] = 2.0 ** 8
    small = vsc.clone()
    vsc.copy_(large)
    want_large = call()
    vsc.copy_(small)
    want = call()
    assert not torch.equal(want, want_large)
    out = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out=out)
    side = torch.cuda.Stream()
    for scales, expect in ((small, want), (large, want_large), (small, want), (large, want_large)):
        vsc.copy_(scales)
        g.replay()
        assert torch.equal(out, expect)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, expect)
