"""The 8-bit cache's numpy restatement and the refusals of its entry points (no GPU)."""

import ctypes

import numpy as np
import pytest
import torch

import infrared_b200 as irb
from infrared_b200 import _lib, ops
from oracle import kv_q8_np as q8


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_encode_agrees_with_the_types(fmt):
    x = np.concatenate([np.linspace(-500, 500, 4001), np.random.default_rng(0).normal(size=4000),
                        2.0 ** np.arange(-14, 9), 0.5 * 2.0 ** np.arange(-14, 9) * 17 / 8])
    t = torch.from_numpy(x.astype(np.float32))
    if fmt == "e4m3":
        want = t.clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    else:
        want = t.round().clamp(-127, 127).numpy()
    np.testing.assert_array_equal(q8.encode(x.astype(np.float32), fmt), want)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scale_is_the_smallest_power_of_two(fmt):
    top = q8.LARGEST[fmt]
    for amax in (0.0, 1e-45, 1e-30, 0.3, top, np.nextafter(top, 1e9), 2 * top, 6e4, 3e38):
        s = q8.scale_for(amax, fmt)
        assert amax <= top * s and np.log2(s) == int(np.log2(s))
        assert s == 2.0 ** -126 or amax > top * s / 2


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_block_filled_token_by_token_has_the_scale_of_its_rows(fmt):
    rng = np.random.default_rng(3)
    bs, h, d = 4, 2, 8
    rows = rng.normal(size=(bs, h, d)) * np.array([0.01, 3.0, 0.1, 90.0])[:, None, None]
    codes, scale = np.full((2 * bs, h, d), 7.0), np.full((2, h), 2.0 ** 30)
    for i in range(bs):
        q8.write(codes, scale, rows[i:i + 1], [bs + i], bs, fmt)
    once, s1 = np.zeros((2 * bs, h, d)), np.zeros((2, h))
    q8.write(once, s1, rows, range(bs, 2 * bs), bs, fmt)
    np.testing.assert_array_equal(scale[1], s1[1])
    assert (scale[0] == 2.0 ** 30).all() and (codes[:bs] == 7.0).all()
    # a code is off by half a unit of the final scale, plus half a unit of each
    # smaller scale it went through: less than one unit in all
    unit = (2.0 ** -3 * np.abs(rows).max() if fmt == "e4m3" else s1[1].max())
    assert np.abs(codes[bs:] * scale[1][None, :, None] - rows).max() < unit


def _decode_shape(**kw):
    base = dict(batch=2, num_heads=28, num_kv_heads=4, head_dim=128, block_size=16, max_blocks=8,
                bt_stride=8, q_stride=28 * 128, out_stride=28 * 128, num_slots=1024, scale=0.088,
                dtype=1, flags=0)
    return _lib.DecodeShape(**{**base, **kw})


@pytest.mark.parametrize("change,fmt,status", [
    ({"head_dim": 96}, 1, _lib.IR_ERR_UNSUPPORTED),
    ({"num_kv_heads": 3}, 1, _lib.IR_ERR_INVALID_ARG),
    ({"num_heads": 68}, 2, _lib.IR_ERR_UNSUPPORTED),      # group of 17
    ({"num_slots": 100}, 2, _lib.IR_ERR_INVALID_ARG),
    ({"dtype": 9}, 1, _lib.IR_ERR_INVALID_ARG),
    ({"flags": 1}, 1, _lib.IR_ERR_INVALID_ARG),
    ({}, 0, _lib.IR_ERR_INVALID_ARG),
    ({}, 3, _lib.IR_ERR_INVALID_ARG),
])
def test_decode_q8_refusals(change, fmt, status):
    lib = _lib.load()
    s = _decode_shape(**change)
    rc = lib.ir_paged_decode_q8(None, None, None, None, None, None, fmt, None, None,
                                ctypes.byref(s), None, 0, None, None)
    assert rc == status, lib.ir_last_error()
    assert lib.ir_paged_decode_q8_workspace_size(ctypes.byref(s), fmt) == 0


def test_write_and_gather_refusals():
    lib = _lib.load()

    def write(n=4, hkv=2, d=64, bs=16, slots=64, dtype=1, fmt=1, stride=128):
        return lib.ir_cache_write_q8(None, None, stride, stride, None, None, None, None, None, n,
                                     hkv, d, bs, slots, dtype, fmt, None, 0, None, None)

    def gather(n=4, hkv=2, d=64, bs=16, slots=64, dtype=1, fmt=1):
        return lib.ir_cache_gather_q8(None, None, None, None, n, hkv, d, bs, slots, dtype, fmt,
                                      None, None)

    assert write(n=0) == _lib.IR_OK and gather(n=0) == _lib.IR_OK
    for call in (write, gather):
        assert call() == _lib.IR_ERR_INVALID_ARG                  # null pointers
        assert call(dtype=7) == _lib.IR_ERR_INVALID_ARG
        assert call(fmt=0) == _lib.IR_ERR_INVALID_ARG
        assert call(slots=65) == _lib.IR_ERR_INVALID_ARG
        assert call(n=-1) == _lib.IR_ERR_INVALID_ARG
        assert call(d=80) == _lib.IR_ERR_UNSUPPORTED
        assert call(n=2 ** 31) == _lib.IR_ERR_UNSUPPORTED
    assert write(stride=100) == _lib.IR_ERR_INVALID_ARG
    assert write(bs=2048, slots=2048) == _lib.IR_ERR_UNSUPPORTED
    assert lib.ir_cache_write_q8_workspace_size(64, 1024, 16) == 0
    assert lib.ir_cache_write_q8_workspace_size(5000, 65536, 16) > 0


def test_prefill_q8_and_norm_refusals():
    lib = _lib.load()
    s = _lib.PrefillShape(num_seqs=1, total_q=4, num_heads=4, num_kv_heads=2, head_dim=64,
                          block_size=16, max_blocks=2, bt_stride=2, q_stride=256, out_stride=256,
                          num_slots=64, scale=0.1, dtype=1)
    call = lambda fmt: lib.ir_paged_prefill_q8(  # noqa: E731
        None, None, None, None, None, None, fmt, None, None, None, ctypes.byref(s), None, 0, None,
        None)
    assert call(5) == _lib.IR_ERR_INVALID_ARG
    assert call(1) == _lib.IR_ERR_INVALID_ARG                     # null pointers
    assert lib.ir_paged_prefill_q8_plan(ctypes.byref(s), 7, None) == _lib.IR_ERR_INVALID_ARG
    s.num_slots = 70
    assert call(1) == _lib.IR_ERR_INVALID_ARG

    def norm(d=64, n=3, dtype=1, eps=1e-6, stride=256, rs=64):
        return lib.ir_qk_norm_rope(None, None, None, None, stride, stride, stride, stride, None,
                                   None, None, None, rs, eps, n, 4, 2, d, dtype, None)

    assert norm(n=0) == _lib.IR_OK
    assert norm() == _lib.IR_ERR_INVALID_ARG
    assert norm(d=96) == _lib.IR_ERR_UNSUPPORTED
    assert norm(dtype=4) == _lib.IR_ERR_INVALID_ARG
    assert norm(eps=-1.0) == _lib.IR_ERR_INVALID_ARG
    assert norm(eps=float("nan")) == _lib.IR_ERR_INVALID_ARG
    assert norm(stride=100) == _lib.IR_ERR_INVALID_ARG
    assert norm(rs=32) == _lib.IR_ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    pool = torch.zeros(32, 2, 64, dtype=torch.int8)
    sc = torch.zeros(2, 2)
    k = torch.zeros(1, 2, 64)
    slots = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError):
        irb.cache_write_q8(k, k, pool, pool, sc, sc, slots, 16)
    with pytest.raises(ValueError):
        irb.cache_gather_q8(pool, sc, slots, 16, torch.float32)
    with pytest.raises(ValueError):
        irb.qk_norm_rope(k, k, None, None, k[:, 0], k[:, 0], 1e-6)
    with pytest.raises(irb.UnsupportedShape):
        ops.kv_format(torch.uint8)


class _FakeLib:
    """Entry points that record which device was current when they were called."""

    def __init__(self, now):
        self.now, self.seen = now, []

    def __getattr__(self, name):
        def call(*args):
            self.seen.append((name, self.now[-1]))
            return 4096 if name.endswith("_workspace_size") else 0
        return call


def test_sizes_are_asked_of_the_tensors_device(monkeypatch):
    """A call on device 1 while device 0 is current: plans, workspace sizes and
    launches all see device 1 (sizes follow the device's SM count)."""
    now = [0]

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            now.append(self.dev)

        def __exit__(self, *exc):
            now.pop()

    lib = _FakeLib(now)
    monkeypatch.setattr(ops, "_dev_index", lambda t: 1)
    monkeypatch.setattr(ops, "_plan_device", lambda t: 1)
    monkeypatch.setattr(ops, "_current_device", lambda: now[-1])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_err_ptr", lambda dev: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    for plans in ("_decode_q8_plans", "_prefill_q8_plans"):
        monkeypatch.setattr(ops, plans, ops._Plans())
    pool = torch.zeros(64, 2, 64, dtype=torch.int8)
    sc, q = torch.zeros(4, 2), torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    bt, ctx = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    qs = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    ops.decode_plan_q8(q, pool, bt, 16)
    ops.prefill_plan_q8(q, pool, bt, qs, 16)
    irb.paged_decode_q8(q, pool, pool, sc, sc, bt, ctx, 0.1, 16)
    irb.paged_prefill_q8(q, pool, pool, sc, sc, bt, ctx, qs, 0.1, 16)
    assert [name for name, _ in lib.seen] == [
        "ir_paged_decode_q8_plan", "ir_paged_decode_q8_workspace_size",
        "ir_paged_prefill_q8_plan", "ir_paged_prefill_q8_workspace_size",
        "ir_paged_decode_q8_workspace_size", "ir_paged_decode_q8",
        "ir_paged_prefill_q8_workspace_size", "ir_paged_prefill_q8"]
    assert all(dev == 1 for _, dev in lib.seen) and now == [0]
