"""Host side of the paged-cache operators, without a GPU: rotation tables, the division by page sizes, refusals of the C ABI."""
import ctypes
import math

import pytest
import torch

from boostr_b200 import _cabi, attention
from boostr_b200.format import QuantError


def test_rope_tables_plain():
    cos, sin = attention.rope_tables(50, 16, base=500.0, device="cpu")
    for p in (0, 1, 49):
        for i in range(8):
            a = p * 500.0 ** (-2 * i / 16)
            assert abs(float(cos[p, i]) - math.cos(a)) < 1e-7 and abs(float(sin[p, i]) - math.sin(a)) < 1e-7


def test_rope_tables_scaled():
    n, r, base = 64, 32, 10000.0
    inv = [base ** (-2 * i / r) for i in range(r // 2)]

    def angles(**s):  # of position 1 (all below pi)
        cos, sin = attention.rope_tables(n, r, base, s, device="cpu")
        return torch.atan2(sin[1].double(), cos[1].double()).tolist(), float(torch.hypot(cos[1], sin[1]).max())

    a, _ = angles(type="linear", factor=4.0)
    assert all(abs(x - y / 4) < 1e-6 for x, y in zip(a, inv))
    a, _ = angles(type="ntk", factor=4.0)
    assert abs(a[0] - inv[0]) < 1e-6 and abs(a[-1] - inv[-1] / 4) < 1e-6  # the fastest kept, the slowest divided
    a, _ = angles(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_positions=256)
    for x, y in zip(a, inv):
        turns = 256 * y / (2 * math.pi)
        want = y if turns >= 4 else y / 8 if turns <= 1 else y * ((turns - 1) / 3) + y / 8 * (1 - (turns - 1) / 3)
        assert abs(x - want) < 1e-6
    a, gain = angles(type="yarn", factor=16.0, original_positions=256)
    assert abs(gain - (0.1 * math.log(16.0) + 1)) < 1e-6
    assert abs(a[0] - inv[0]) < 1e-6 and abs(a[-1] - inv[-1] / 16) < 1e-6
    assert all(y / 16 - 1e-6 <= x <= y + 1e-6 for x, y in zip(a, inv))
    for bad in ({"type": "other"}, {"type": "linear", "factor": 0.0}):
        with pytest.raises(QuantError):
            attention.rope_tables(n, r, base, bad, device="cpu")
    with pytest.raises(QuantError):
        attention.rope_tables(n, 3, device="cpu")


def test_division_by_page_sizes():
    """The kernels' n / d by a multiplication (FastDiv), restated: all small divisors, and the ends of the range."""
    for d in list(range(1, 300)) + [1023, 1024, 1025, 65535, (1 << 31) - 1]:
        l = 0
        while (1 << l) < d:
            l += 1
        m = ((((1 << l) - d) << 32) // d + 1) & 0xFFFFFFFF
        for n in [0, 1, d - 1, d, d + 1, 7 * d - 1, 7 * d, (1 << 31) - 1, (1 << 31) - 2, ((1 << 31) - 1) // d * d, ((1 << 31) - 1) // d * d - 1]:
            if 0 <= n < 1 << 31:
                s = ((m * n) >> 32) + n
                assert s < 1 << 32 and s >> l == n // d, (n, d)


def test_cabi_refusals():
    L = _cabi.lib()
    p = ctypes.c_void_p(0x10000)

    def cache(**o):
        f = dict(k=p, v=p, dtype=_cabi.DT_BF16, pages=4, page_size=16, kv_heads=2, head_dim=64)
        f.update(o)
        return _cabi.PagedCache(f["k"], f["v"], f["dtype"], f["pages"], f["page_size"], f["kv_heads"], f["head_dim"],
                                (ctypes.c_int64 * 3)(2048, 128, 64), (ctypes.c_int64 * 3)(*f.get("vs", (2048, 128, 64))))

    def decode(c, q=p, qt=_cabi.DT_BF16, row=256, hq=4, width=3, scale=1.0, ot=_cabi.DT_BF16, n=2):
        return L.b200q_paged_decode(q, qt, row, 64, n, hq, c, p, width, width, p, scale, 0, 0, p, ot, None, None, 0, None)

    assert decode(cache(), n=0) == _cabi.OK
    for rc, want in [(decode(cache(dtype=_cabi.DT_F32)), _cabi.ERR_UNSUPPORTED_DTYPE), (decode(cache(pages=0)), _cabi.ERR_BAD_SHAPE),
                     (decode(cache(head_dim=60)), _cabi.ERR_BAD_SHAPE), (decode(cache(head_dim=512)), _cabi.ERR_BAD_SHAPE),
                     (decode(cache(k=ctypes.c_void_p(0x10008))), _cabi.ERR_INVALID_ARG), (decode(cache(vs=(2048, 132, 64))), _cabi.ERR_BAD_SHAPE),
                     (decode(cache(), q=None), _cabi.ERR_INVALID_ARG), (decode(cache(), qt=_cabi.DT_F16), _cabi.ERR_UNSUPPORTED_DTYPE),
                     (decode(cache(), row=255), _cabi.ERR_INVALID_ARG), (decode(cache(), hq=3), _cabi.ERR_BAD_SHAPE),
                     (decode(cache(), width=0), _cabi.ERR_BAD_SHAPE), (decode(cache(), scale=math.nan), _cabi.ERR_INVALID_ARG),
                     (decode(cache(), ot=_cabi.DT_F64), _cabi.ERR_UNSUPPORTED_DTYPE)]:
        assert rc == want, L.b200q_last_error()
    h = _cabi.Heads(p, 256, 64)
    rope = lambda c, rot=64, dt=0: L.b200q_rope_append(h, h, h, dt, 3, 4, p, p, p, 10, rot, 0, None, None, 1e-5, c, p, p, 0, None)  # noqa: E731
    assert rope(cache(), rot=66) == _cabi.ERR_BAD_SHAPE and rope(cache(), rot=3) == _cabi.ERR_BAD_SHAPE
    assert rope(cache(), dt=_cabi.DT_F64) == _cabi.ERR_UNSUPPORTED_DTYPE
    assert L.b200q_paged_slots(p, p, 0, p, 3, 3, 16, p, 9, p, p, p, p, p, 4, p, None) == _cabi.ERR_BAD_SHAPE
    assert L.b200q_paged_slots(p, p, 2, p, 3, 3, 0, p, 9, p, p, p, p, p, 4, p, None) == _cabi.ERR_BAD_SHAPE
    assert L.b200q_paged_slots(p, None, 2, p, 3, 3, 16, p, 9, p, p, p, p, p, 4, p, None) == _cabi.ERR_INVALID_ARG
    assert L.b200q_paged_prompt(p, _cabi.DT_F32, 256, 64, 2, 4, p, 1, cache(), p, 3, 3, p, 1.0, 0, 0, p, 0, None, None, 0, None) == _cabi.ERR_UNSUPPORTED_DTYPE
