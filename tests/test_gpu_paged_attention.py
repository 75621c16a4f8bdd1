"""Attention from a paged cache (``boostr_b200.attention``) against plain 64-bit forms.

Tolerances follow from the roundings that the operators state.  With u the unit roundoff of the cache's type (2^-8 bf16, 2^-11
f16), A = sum_j p_j |v_j| and D = max_j scale sum_e |q_e k_je| of a row:

* weights are rounded to the cache's type (16-bit queries) or kept to 2^-15 (f32 queries), each against A;
* scores carry the f32 sums' error, head_dim 2^-24 D, and with f32 queries the split's 2^-16 D; a weight changes by twice that;
* the exponentials and the remaining f32 sums stay within 2^-17 (one token) and 2^-12 (prompts: a cubic in place of the function);
* the result is rounded once to the output's type."""
import math

import pytest

from boostr_b200 import _cabi, ops
from boostr_b200.format import QuantError

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def attention():
    from boostr_b200 import attention as a

    return a


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def make_cache(g, lens, page, hk, d, dtype, layout="tokens", spare=3):
    """A cache whose unused places hold NaN and infinities, and block tables in random order (-1 behind their pages)."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    if layout == "heads":
        both = torch.randn(2, pages, hk, page, d, device="cuda", generator=g).to(dtype).transpose(2, 3)
    elif layout == "joint":  # keys and values side by side in one tensor
        both = torch.randn(pages, page, 2, hk, d, device="cuda", generator=g).to(dtype).permute(2, 0, 1, 3, 4)
    else:
        both = torch.randn(2, pages, page, hk, d, device="cuda", generator=g).to(dtype)
    k, v = both[0], both[1]
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for j in range(n):
            used[table[b, j].long(), : min(page, lens[b] - j * page)] = True
    k[~used] = math.nan
    v[~used] = math.inf
    v[..., ::2, :][~used] = math.nan
    return k, v, table


def visible(pos, n, window, sinks):
    key = torch.arange(n, device="cuda")
    m = key <= pos[:, None]
    if window:
        m &= (pos[:, None] - key < window) | (key < sinks)
    return m


def reference(q, pos, b, k, v, table, length, scale, window, sinks):
    """Rows q [n, hq, d] of request b at positions pos: out, lse, A and D (see above), all f64."""
    n, hq, d = q.shape
    page, hk = k.shape[1], k.shape[2]
    idx = table[b, : -(-length // page)].long()
    kk, vv = (c[idx].flatten(0, 1)[:length].double() for c in (k, v))
    seen = visible(pos, length, window, sinks)
    kk, vv = (torch.where(seen.any(0)[:, None, None], c, 0.0) for c in (kk, vv))
    kh, vh = (c.repeat_interleave(hq // hk, 1) for c in (kk, vv))
    s = torch.einsum("nhd,khd->nhk", q.double(), kh) * scale
    big = torch.einsum("nhd,khd->nhk", q.double().abs(), kh.abs()) * abs(scale)
    s.masked_fill_(~seen[:, None], -math.inf)
    big.masked_fill_(~seen[:, None], 0.0)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen[:, None], torch.exp(s - lse[..., None]), 0.0)
    return torch.einsum("nhk,khd->nhd", p, vh), lse, torch.einsum("nhk,khd->nhd", p, vh.abs()), big.amax(-1) if length else torch.zeros_like(lse)


def check(got, lse, want, q, out_dtype, cache_dtype, prompt):
    out, ref_lse, A, D = want
    d = q.shape[-1]
    c_s = d * 2.0 ** -24 + (2.0 ** -16 if q.dtype == F32 else 0.0)
    c_p = 2.0 ** -15 if q.dtype == F32 else U[cache_dtype]
    c_e = 2.0 ** -12 if prompt else 2.0 ** -17
    tol = A * (c_p + c_e + 2 * c_s * D[..., None]) + U[out_dtype] * out.abs() * 1.01 + 1e-30
    if out_dtype == F16:
        tol = tol + 2.0 ** -25  # the spacing of its subnormals
    bad = ~((got.double() - out).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - out).abs() / tol).nan_to_num(math.inf).max()):.2f} of the tolerance"
    if lse is not None:
        fine = ref_lse > -math.inf
        assert torch.equal(lse > -math.inf, fine)
        bad = fine & ~((lse.double() - ref_lse).abs() <= c_e + c_s * D + 2.0 ** -22 * ref_lse.abs())
        assert not bad.any()


# ------------------------------------------------------------------------------------------------------------------- decode

DECODE = [
    # lens, page, hq, hk, d, window, sinks, q type, cache type, out type, layout
    ([1], 16, 1, 1, 8, 0, 0, BF16, BF16, BF16, "tokens"),
    ([1, 0, 2, 17], 16, 4, 1, 64, 0, 0, F32, BF16, F32, "tokens"),
    ([517], 16, 32, 8, 128, 0, 0, BF16, BF16, BF16, "tokens"),
    ([300, 0, 0, 65, 64, 63], 16, 32, 8, 128, 0, 0, F32, BF16, F32, "heads"),
    ([1000, 1, 333], 1, 8, 8, 64, 0, 0, F16, F16, F16, "tokens"),
    ([700, 129], 7, 6, 2, 80, 0, 0, BF16, BF16, F32, "joint"),
    ([257, 31], 32, 15, 5, 96, 0, 0, F32, F16, F16, "joint"),
    ([2050], 64, 16, 1, 256, 0, 0, BF16, BF16, BF16, "heads"),
    ([90, 400], 16, 48, 2, 128, 0, 0, F16, F16, F32, "tokens"),     # 24 query heads to a key-value head
    ([60, 3], 16, 71, 1, 40, 0, 0, F32, BF16, BF16, "tokens"),  # 71 of them
    ([5000, 40, 1024, 1029], 32, 16, 2, 64, 1024, 4, F16, F16, F16, "tokens"),
    ([5000, 3, 0], 16, 8, 8, 128, 1, 0, BF16, BF16, BF16, "tokens"),   # only the token itself
    ([5000, 700], 16, 8, 4, 128, 100, 130, F32, BF16, F32, "heads"),   # more sinks than window, both ends inside pages
    ([200, 90], 128, 8, 4, 128, 1000, 50, BF16, BF16, BF16, "tokens"), # a window that hides nothing
    ([40000], 16, 4, 1, 128, 0, 0, F32, BF16, F32, "tokens"),          # split over the length and joined
    ([70001, 5, 30000], 64, 32, 8, 128, 0, 0, BF16, BF16, BF16, "tokens"),
]


@pytest.mark.parametrize("i", range(len(DECODE)))
def test_decode(attention, i):
    lens, page, hq, hk, d, window, sinks, qt, ct, ot, layout = DECODE[i]
    g = _gen(100 + i)
    k, v, table = make_cache(g, lens, page, hk, d, ct, layout)
    q = _randn(g, len(lens), hq, d, dtype=F32).mul_(1.5).to(qt)
    for scale in (None, 0.3):
        out, lse = attention.paged_decode(q, k, v, table, _ints(lens), scale=scale, window=window, sinks=sinks, out_dtype=ot, return_lse=True)
        ops.check_device_status()
        sc = d ** -0.5 if scale is None else scale
        for b, n in enumerate(lens):
            if n == 0:
                assert not out[b].any() and (lse[b] == -math.inf).all()
                continue
            want = reference(q[b:b + 1], _ints([n - 1]), b, k, v, table, n, sc, window, sinks)
            check(out[b:b + 1], lse[b:b + 1], want, q, ot, ct, False)
    again = attention.paged_decode(q, k, v, table, _ints(lens), scale=0.3, window=window, sinks=sinks, out_dtype=ot)
    assert torch.equal(out.nan_to_num(0), again.nan_to_num(0)), "two calls differ"


@pytest.mark.parametrize("requests", [1, 37, 300, 1500])
def test_decode_many_requests(attention, requests):
    g = _gen(requests)
    lens = torch.randint(0, 200, (requests,), generator=g, device="cuda").tolist()
    hq, hk, d = 8, 2, 64
    k, v, table = make_cache(g, lens, 16, hk, d, BF16)
    q = _randn(g, requests, hq, d, dtype=BF16)
    out = attention.paged_decode(q, k, v, table, _ints(lens))
    ops.check_device_status()
    for b in list(range(0, requests, max(1, requests // 40))) + [requests - 1]:
        if lens[b]:
            check(out[b:b + 1], None, reference(q[b:b + 1], _ints([lens[b] - 1]), b, k, v, table, lens[b], d ** -0.5, 0, 0), q, BF16, BF16, False)
        else:
            assert not out[b].any()


def test_decode_infinite_scores_and_values(attention):
    """Peaked softmax over a huge range, and keys whose scores are minus infinity, weigh nothing."""
    g = _gen(5)
    lens, d = [400], 128
    k, v, table = make_cache(g, lens, 16, 2, d, F16)
    q = (_randn(g, 1, 8, d) * 40).to(F16)
    page = table[0, 3].long()
    k[page, 5] = 0
    k[page, 5, :, 0] = -math.inf
    v[page, 5] = 3.0
    q[..., 0] = q[..., 0].abs() + 1
    out, lse = attention.paged_decode(q, k, v, table, _ints(lens), return_lse=True)
    ref = k.clone()
    ref[page, 5, :, 0] = -65504.0  # a finite key of the same weight, none
    check(out, None, reference(q, _ints([399]), 0, ref, v, table, 400, d ** -0.5, 0, 0)[:3] + (torch.full((1, 8), 500.0, device="cuda"),), q, F16, F16, False)


def test_output_over_the_queries_is_refused(attention):
    g = _gen(7)
    k, v, table = make_cache(g, [40, 9], 16, 2, 64, BF16)
    q = _randn(g, 2, 8, 64, dtype=BF16)
    pool = torch.empty(3, 8, 64, dtype=BF16, device="cuda")
    pool[:2] = q
    for out in (pool[:2], pool[1:]):
        with pytest.raises(_cabi.B200QError, match="must not overlap"):
            attention.paged_decode(pool[:2], k, v, table, _ints([40, 9]), out=out)
        with pytest.raises(_cabi.B200QError, match="must not overlap"):
            attention.paged_prompt(pool[:2], _ints([0, 1, 2]), k, v, table, _ints([40, 9]), out=out)
    want = attention.paged_decode(q[:1], k, v, table[:1], _ints([40]))
    assert torch.equal(attention.paged_decode(pool[:1], k, v, table[:1], _ints([40]), out=pool[1:2]), want)  # next to them


@pytest.mark.parametrize("rows", [1, 5, 700])
def test_prompt_of_no_request_is_zero(attention, rows):
    g = _gen(8)
    k, v, table = make_cache(g, [40], 16, 2, 64, BF16)
    out = torch.ones(rows, 8, 64, dtype=BF16, device="cuda")
    _, lse = attention.paged_prompt(_randn(g, rows, 8, 64, dtype=BF16), _ints([0]), k, v, table[:0], _ints([]), out=out, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


def test_decode_strided_queries_and_given_output(attention):
    g = _gen(6)
    lens = [333, 20]
    k, v, table = make_cache(g, lens, 16, 4, 64, BF16)
    rows = _randn(g, 2, 16 * 64 + 2 * 4 * 64, dtype=BF16)
    q = rows[:, : 16 * 64].view(2, 16, 64)
    want = attention.paged_decode(q.contiguous(), k, v, table, _ints(lens))
    assert torch.equal(attention.paged_decode(q, k, v, table, _ints(lens)), want)
    one = q[:1, :1].expand(2, 16, 64)  # one head for all: copied
    assert torch.equal(attention.paged_decode(one, k, v, table, _ints(lens)), attention.paged_decode(one.contiguous(), k, v, table, _ints(lens)))
    cu = _ints([0, 1, 2])
    assert torch.equal(attention.paged_prompt(one, cu, k, v, table, _ints(lens)), attention.paged_prompt(one.contiguous(), cu, k, v, table, _ints(lens)))
    flat = q[0].reshape(-1).as_strided((1, 16, 64), (0, 64, 1))  # one row whose stride says nothing
    assert torch.equal(attention.paged_prompt(flat, cu[:2], k, v, table[:1], _ints(lens[:1])), attention.paged_prompt(q[:1], cu[:2], k, v, table[:1], _ints(lens[:1])))
    single = rows.new_zeros(1, 16 * 64 + 5)[:, : 16 * 64].view(1, 16, 64)  # one row of an odd stride
    single.copy_(q[:1])
    assert torch.equal(attention.paged_decode(single, k, v, table[:1], _ints(lens[:1])), want[:1])
    assert torch.equal(attention.paged_prompt(single, cu[:2], k, v, table[:1], _ints(lens[:1])), attention.paged_prompt(q[:1].contiguous(), cu[:2], k, v, table[:1], _ints(lens[:1])))
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads before tokens in memory
    assert torch.equal(attention.paged_decode(turned, k, v, table, _ints(lens)), want)
    assert torch.equal(attention.paged_prompt(turned, cu, k, v, table, _ints(lens)), attention.paged_prompt(q, cu, k, v, table, _ints(lens)))
    odd = _randn(g, 2, 16, 65, dtype=BF16)
    odd[..., 1:] = q
    assert torch.equal(attention.paged_decode(odd[..., 1:], k, v, table, _ints(lens)), want)  # unaligned: copied
    out = torch.empty_like(want)
    assert attention.paged_decode(q, k, v, table, _ints(lens), out=out) is out and torch.equal(out, want)
    wide = torch.full((2, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    assert torch.equal(attention.paged_decode(q, k, v, wide[:, : table.shape[1] + 3], _ints(lens)), want)
    f32 = attention.paged_decode(q.float(), k, v, table, _ints(lens), out=torch.empty(2, 16, 64, device="cuda"))
    assert f32.dtype == F32 and (f32 - want.float()).abs().max() < 2e-2


def test_decode_in_another_stream_and_in_a_graph(attention):
    g = _gen(7)
    lens = [20000, 3, 700]
    k, v, table = make_cache(g, lens, 16, 8, 128, BF16)
    q = _randn(g, 3, 32, 128, dtype=BF16)
    n = _ints(lens)
    want = attention.paged_decode(q, k, v, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [attention.paged_decode(q, k, v, table, n) for _ in range(3)]
    here = [attention.paged_decode(q, k, v, table, n) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got + here)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.paged_decode(q, k, v, table, n, out=out)
    for m in ([20000, 3, 700], [500, 3, 0], [19999, 1, 64]):  # the lengths change between replays
        n.copy_(_ints(m))
        graph.replay()
        eager = attention.paged_decode(q, k, v, table, n)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_decode_offsets_beyond_32_bits(attention):
    """Pages more than 2^31 elements into the cache."""
    g = _gen(8)
    page, hk, d = 64, 8, 128
    pages = (1 << 31) // (page * hk * d) + 40
    k, v = (torch.empty(pages, page, hk, d, dtype=BF16, device="cuda") for _ in range(2))
    lens = [1000]
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.cat([torch.tensor([pages - 1 - i for i in range(8)], device="cuda"), order[order < pages - 8][:8]]).to(torch.int32)[None]
    for t in (k, v):
        t[table[0].long()] = _randn(g, 16, page, hk, d, dtype=BF16)
    q = _randn(g, 1, 32, d, dtype=BF16)
    out = attention.paged_decode(q, k, v, table, _ints(lens))
    check(out, None, reference(q, _ints([999]), 0, k, v, table, 1000, d ** -0.5, 0, 0), q, BF16, BF16, False)
    cu = _ints([0, 100])
    q = _randn(g, 100, 32, d, dtype=BF16)
    out = attention.paged_prompt(q, cu, k, v, table, _ints(lens))
    check(out, None, reference(q, torch.arange(900, 1000, device="cuda"), 0, k, v, table, 1000, d ** -0.5, 0, 0), q, BF16, BF16, True)


# ------------------------------------------------------------------------------------------------------------------- prompts

PROMPT = [
    # (tokens before, new tokens) of each request, page, hq, hk, d, window, sinks, type, out type, layout, rows behind the last
    ([(0, 1)], 16, 1, 1, 8, 0, 0, BF16, BF16, "tokens", 0),
    ([(0, 33)], 16, 32, 8, 128, 0, 0, BF16, BF16, "tokens", 0),
    ([(0, 512)], 16, 8, 2, 128, 0, 0, BF16, BF16, "tokens", 0),
    ([(0, 300), (5, 0), (700, 129), (0, 1), (63, 64)], 16, 8, 2, 128, 0, 0, BF16, F32, "heads", 5),
    ([(0, 257), (100, 3)], 1, 4, 4, 64, 0, 0, F16, F16, "tokens", 0),
    ([(17, 200), (0, 77)], 7, 6, 2, 80, 0, 0, BF16, BF16, "joint", 0),
    ([(1000, 130)], 32, 15, 5, 96, 0, 0, F16, F16, "joint", 3),
    ([(40, 600)], 64, 16, 1, 256, 0, 0, BF16, BF16, "heads", 0),
    ([(0, 90), (300, 20)], 16, 48, 2, 128, 0, 0, F16, F32, "tokens", 0),  # 24 query heads to a key-value head
    ([(9, 45)], 16, 71, 1, 40, 0, 0, BF16, BF16, "tokens", 0),
    ([(3000, 400), (0, 1500), (0, 10)], 32, 16, 2, 64, 1024, 4, F16, F16, "tokens", 0),
    ([(2000, 300), (0, 5)], 16, 8, 8, 128, 1, 0, BF16, BF16, "tokens", 0),
    ([(2000, 300), (50, 500)], 16, 8, 4, 128, 100, 130, BF16, BF16, "heads", 0),
    ([(0, 700)], 128, 8, 4, 128, 130, 0, BF16, BF16, "tokens", 0),
    ([(0, 1500)], 16, 4, 4, 128, 0, 0, BF16, BF16, "tokens", 0),
    ([(6000, 700)], 16, 4, 1, 128, 0, 0, BF16, BF16, "tokens", 0),
    # few rows over many keys: the keys are split and joined
    ([(20000, 3)], 16, 32, 8, 128, 0, 0, BF16, BF16, "tokens", 0),
    ([(30000, 1), (9000, 40), (0, 5), (100, 0)], 64, 8, 2, 64, 0, 0, F16, F32, "heads", 2),
    ([(7000, 70)], 16, 4, 1, 256, 0, 0, BF16, BF16, "tokens", 0),
    ([(9000, 20), (400, 30)], 7, 6, 1, 80, 0, 0, F16, F16, "joint", 0),
    ([(50000, 9)], 32, 16, 2, 128, 3000, 20, BF16, BF16, "heads", 0),
]


@pytest.mark.parametrize("i", range(len(PROMPT)))
def test_prompt(attention, i):
    shape, page, hq, hk, d, window, sinks, ct, ot, layout, behind = PROMPT[i]
    g = _gen(200 + i)
    lens = [c + n for c, n in shape]
    cu = [0]
    for _, n in shape:
        cu.append(cu[-1] + n)
    k, v, table = make_cache(g, lens, page, hk, d, ct, layout)
    q = _randn(g, cu[-1] + behind, hq, d).mul_(1.5).to(ct)
    for scale in (None, 0.3):
        out, lse = attention.paged_prompt(q, _ints(cu), k, v, table, _ints(lens), scale=scale, window=window, sinks=sinks, out_dtype=ot, return_lse=True)
        ops.check_device_status()
        sc = d ** -0.5 if scale is None else scale
        for b, (c, n) in enumerate(shape):
            if n:
                rows = slice(cu[b], cu[b + 1])
                want = reference(q[rows], torch.arange(c, c + n, device="cuda"), b, k, v, table, lens[b], sc, window, sinks)
                check(out[rows], lse[rows], want, q, ot, ct, True)
        assert not out[cu[-1]:].any() and (lse[cu[-1]:] == -math.inf).all()
    again = attention.paged_prompt(q, _ints(cu), k, v, table, _ints(lens), scale=0.3, window=window, sinks=sinks, out_dtype=ot)
    assert torch.equal(out, again), "two calls differ"


def test_prompt_rows_without_keys(attention):
    """More rows than tokens (an inconsistent padded request): the rows before the first token see nothing."""
    g = _gen(9)
    k, v, table = make_cache(g, [5, 0], 16, 2, 64, BF16)
    q = _randn(g, 12, 4, 64, dtype=BF16)
    out, lse = attention.paged_prompt(q, _ints([0, 8, 12]), k, v, table, _ints([5, 0]), return_lse=True)
    assert not out[:3].any() and (lse[:3] == -math.inf).all() and not out[8:].any() and (lse[8:] == -math.inf).all()
    check(out[3:8], lse[3:8], reference(q[3:8], torch.arange(5, device="cuda"), 0, k, v, table, 5, 0.125, 0, 0), q, BF16, BF16, True)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_prompt_values_that_a_row_does_not_see(attention, bad):
    """A value that is not a finite number reaches the rows that see its token, and no others."""
    g = _gen(10)
    n, d = 300, 128
    k, v, table = make_cache(g, [n], 16, 2, d, BF16)
    v[table[0, 150 // 16].long(), 150 % 16, 1, 7] = bad
    q = _randn(g, n, 8, d, dtype=BF16)
    for window, sinks in ((0, 0), (40, 3)):
        out = attention.paged_prompt(q, _ints([0, n]), k, v, table, _ints([n]), window=window, sinks=sinks)
        hit = torch.zeros(n, 8, d, dtype=torch.bool, device="cuda")
        hit[150: 190 if window else n, 4:, 7] = True
        assert not out[~hit].isnan().any() and not out[~hit].isinf().any()
        assert not out[hit].isfinite().any()
        clean = v.clone()
        clean[table[0, 150 // 16].long(), 150 % 16, 1, 7] = 0
        want = reference(q, torch.arange(n, device="cuda"), 0, k, clean, table, n, d ** -0.5, window, sinks)
        check(out.masked_fill(hit, 0), None, (want[0].masked_fill(hit, 0),) + want[1:], q, BF16, BF16, True)


def test_prompt_agrees_with_decode(attention):
    """The last rows of prompts and a decode step at their positions."""
    g = _gen(11)
    lens = [700, 64, 1]
    k, v, table = make_cache(g, lens, 16, 8, 128, BF16)
    q = _randn(g, 3, 32, 128, dtype=BF16)
    a = attention.paged_prompt(q, _ints([0, 1, 2, 3]), k, v, table, _ints(lens), window=100, sinks=2)
    b = attention.paged_decode(q, k, v, table, _ints(lens), window=100, sinks=2)
    for i, n in enumerate(lens):
        want = reference(q[i:i + 1], _ints([n - 1]), i, k, v, table, n, 128 ** -0.5, 100, 2)
        check(a[i:i + 1], None, want, q, BF16, BF16, True)
        check(b[i:i + 1], None, want, q, BF16, BF16, False)


# ------------------------------------------------------------------------------------------------- refusals and bad indexes


def _fine(attention):
    g = _gen(12)
    k, v, table = make_cache(g, [20, 30], 16, 2, 64, BF16)
    return _randn(g, 2, 4, 64, dtype=BF16), k, v, table, _ints([20, 30])


def test_attention_refusals(attention):
    q, k, v, t, n = _fine(attention)
    cu = _ints([0, 1, 2])
    for f in (lambda *a, **o: attention.paged_decode(*a, **o), lambda q, *a, **o: attention.paged_prompt(q, cu, *a, **o)):
        f(q, k, v, t, n)
        for args, text in [
            ((q.half(), k, v, t, n), "cache's type"),
            ((q[..., :32], k, v, t, n), "queries must be"),
            ((q[:, :3], k, v, t, n), "multiple of 2 heads"),
            ((q[0], k, v, t, n), "queries must be"),
            ((q, k.float(), v.float(), t, n), "BF16 or F16"),
            ((q, k, v[:-1], t, n), "alike"),
            ((q, k, v.half(), t, n), "alike"),
            ((q, k, v, t.long(), n), "block_table"),
            ((q, k, v, t[:1], n), "block_table"),
            ((q, k, v, t, n.long()), "seq_lens"),
            ((q, k, v, t.cpu(), n), "CUDA device"),
            ((q.cpu(), k, v, t, n), "CUDA device"),
            ((q, k.transpose(2, 3).contiguous().transpose(2, 3), v, t, n), "contiguous in the cache"),
        ]:
            with pytest.raises(QuantError, match=text):
                f(*args)
        with pytest.raises(QuantError, match="negative"):
            f(q, k, v, t, n, window=-1)
        with pytest.raises(QuantError, match="negative"):
            f(q, k, v, t, n, window=8, sinks=-1)
        with pytest.raises(QuantError, match="output must be"):
            f(q, k, v, t, n, out_dtype=torch.float64)
        with pytest.raises(QuantError, match="out must be"):
            f(q, k, v, t, n, out=torch.empty(2, 4, 32, dtype=BF16, device="cuda"))
        with pytest.raises(_cabi.B200QError, match="scale must be finite"):
            f(q, k, v, t, n, scale=math.inf)
        big = torch.empty(1, 1, 1, 264, dtype=BF16, device="cuda")
        with pytest.raises(_cabi.B200QError, match="multiple of 8 up to 256"):
            f(torch.empty(2, 1, 264, dtype=BF16, device="cuda"), big, big, t, n)
        odd = torch.empty(4, 16, 2, 68, dtype=BF16, device="cuda")[..., :64]
        with pytest.raises(_cabi.B200QError, match="strides must be multiples of 8"):
            f(q, odd, odd, t, n)
    with pytest.raises(QuantError, match="one row for each request"):
        attention.paged_decode(q[:1], k, v, t, n)
    with pytest.raises(QuantError, match="cu_seqlens"):
        attention.paged_prompt(q, cu[:2], k, v, t, n)
    with pytest.raises(QuantError, match="cache's type"):
        attention.paged_prompt(q.float(), cu, k, v, t, n)
    empty = attention.paged_decode(q[:0], k, v, t[:0], n[:0])
    assert empty.shape == (0, 4, 64)
    assert attention.paged_prompt(q[:0], cu[:1] * 0, k, v, t[:0], n[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("bad", [-1, 1 << 30, "length"])
def test_bad_indexes_are_reported(attention, bad):
    """A page that does not exist, and a length beyond the table, are not followed; other requests keep their results."""
    q, k, v, t, n = _fine(attention)
    for f in (lambda: attention.paged_decode(q, k, v, t, n), lambda: attention.paged_prompt(q, _ints([0, 1, 2]), k, v, t, n)):
        want = f()
        ops.check_device_status()
        keep_t, keep_n = t.clone(), n.clone()
        if bad == "length":
            n[1] = 1 << 20
        else:
            t[1, 1] = bad
        got = f()
        with pytest.raises(_cabi.B200QError, match="out of range"):
            ops.check_device_status()
        assert torch.equal(got[0], want[0])
        t.copy_(keep_t)
        n.copy_(keep_n)
        assert torch.equal(f(), want)
        ops.check_device_status()


# --------------------------------------------------------------------------------------------------------------------- slots


def slots_reference(ctx, new, table, page, free, count, tokens):
    table, width = [list(r) for r in table], len(table[0])
    cu, pos, slot = [0], [], []
    missing = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        for e in range(-(-c // page), -(-(c + n) // page)):
            if e >= width:
                missing += 1
            elif count > 0:
                count -= 1
                table[b][e] = free[count]
            else:
                table[b][e] = -1
                missing += 1
        for i in range(c, c + n):
            pos.append(i)
            p = table[b][i // page] if i // page < width else -1
            slot.append(p * page + i % page if p >= 0 else -1)
        cu.append(cu[-1] + n)
    pad = tokens - len(pos)
    return table, [max(c, 0) + max(n, 0) for c, n in zip(ctx, new)], cu, (pos + [0] * pad)[:tokens], (slot + [-1] * pad)[:tokens], [count, missing]


SLOTS = [
    # requests, ctx up to, new up to, page, width (0: what is needed), pages short, padding
    (1, 0, 1, 16, 0, 0, 0), (1, 100, 0, 16, 0, 0, 3), (64, 500, 1, 16, 0, 0, 0), (300, 50, 40, 7, 0, 0, 11), (257, 400, 300, 64, 0, 5, 0),
    (5, 30, 3000, 1, 0, 0, 0), (40, 100, 100, 16, 6, 0, 0), (40, 100, 100, 16, 6, 20, 1), (1000, 3, 3, 128, 0, 1000, 0), (16384, 5, 2, 4, 0, 0, 0),
    (3, 20, 20, 16, 0, 0, -15),
]


@pytest.mark.parametrize("i", range(len(SLOTS)))
def test_slots(attention, i):
    n, ctx_hi, new_hi, page, width, short, pad = SLOTS[i]
    g = torch.Generator().manual_seed(300 + i)
    ctx = torch.randint(0, ctx_hi + 1, (n,), generator=g).tolist()
    new = torch.randint(0 if n > 1 else new_hi, new_hi + 1, (n,), generator=g).tolist()
    held, want = [-(-c // page) for c in ctx], [-(-(c + m) // page) for c, m in zip(ctx, new)]
    width = width or max(1, max(want))
    order = torch.randperm(sum(want) + 9, generator=g).tolist()
    table = [[-1] * width for _ in range(n)]
    for b in range(n):
        for e in range(min(held[b], width)):
            table[b][e] = order.pop()
    count = max(0, sum(want) - sum(held) - short) if short else len(order)
    tokens = max(0, sum(new) + pad)
    ref = slots_reference(ctx, new, table, page, order, count, tokens)
    t = _ints(table)
    wide = torch.full((n, width + 3), -7, dtype=torch.int32, device="cuda")
    wide[:, :width] = t
    for tab in (t, wide[:, :width]):
        got = attention.paged_slots(_ints(ctx), _ints(new), tab, page, _ints(order), _ints([count]), tokens)
        assert got.block_table is tab
        for name, a, b in zip(got._fields, got, ref):
            assert a.tolist() == b, name
        assert got.slots.dtype == torch.int64
    assert (wide[:, width:] == -7).all()


def test_slots_over_steps(attention):
    """Steps that hand the stack on without the host reading anything, against the count of pages."""
    n, page, pages = 6, 4, 40
    ctx, table = _ints([0] * n), torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(pages, device="cuda").to(torch.int32), _ints([pages])
    for step, new in enumerate([[5, 0, 9, 1, 2, 3], [1] * n, [0, 20, 0, 0, 0, 1], [1] * n]):
        s = attention.paged_slots(ctx, _ints(new), table, page, free, count, sum(new))
        ctx, count = s.seq_lens, s.left[:1].clone()
        assert s.slots.min() >= 0
    used = table[table >= 0].tolist()
    assert len(used) == len(set(used)) == sum(-(-c // page) for c in ctx.tolist()) == pages - int(count)


def test_slots_refusals(attention):
    i = _ints
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    fine = (i([1, 2]), i([1, 1]), table, 16, i([4, 5]), i([2]), 2)
    attention.paged_slots(*fine)
    for at, value, text in [(0, i([1, 2]).long(), "ctx_lens"), (0, table, "1D"), (1, i([1]), "new_lens"), (2, table[:1], "block_table"),
                            (2, table.t(), "block_table"), (4, i([4]).long(), "free_pages"), (5, i([2, 2]), "free_count"), (3, 0, "page size"),
                            (6, -1, "tokens"), (0, i([1, 2]).cpu(), "CUDA device")]:
        args = list(fine)
        args[at] = value
        with pytest.raises(QuantError, match=text):
            attention.paged_slots(*args)
    big = torch.zeros(16385, dtype=torch.int32, device="cuda")
    with pytest.raises(_cabi.B200QError, match="16384 requests"):
        attention.paged_slots(big, big, torch.zeros(16385, 1, dtype=torch.int32, device="cuda"), 16, i([1]), i([1]), 0)


# ---------------------------------------------------------------------------------------------------------------------- rope

ROPE = [
    # tokens, hq, hk, d, rot, interleaved, norms, type, out type, cache type, layout, projection in one tensor
    (1, 32, 8, 128, 128, False, "", F32, F32, BF16, "tokens", True),
    (77, 8, 2, 128, 128, False, "qk", BF16, BF16, BF16, "heads", True),
    (33, 5, 5, 64, 64, True, "qk", F16, F16, F16, "joint", False),
    (50, 20, 5, 80, 32, True, "", F16, F32, F16, "tokens", True),
    (19, 6, 2, 80, 40, False, "q", BF16, F32, BF16, "tokens", True),
    (40, 3, 1, 96, 48, False, "k", F32, BF16, F16, "heads", False),
    (9, 4, 4, 256, 256, False, "qk", F32, F32, BF16, "tokens", False),
    (9, 4, 2, 256, 64, True, "", BF16, F16, BF16, "tokens", True),
    (21, 2, 1, 8, 8, False, "qk", F16, F16, BF16, "tokens", False),
    (21, 2, 1, 8, 2, True, "", F32, F32, BF16, "tokens", False),
    (21, 2, 1, 248, 6, False, "qk", BF16, BF16, BF16, "tokens", False),
    (21, 2, 1, 120, 104, False, "", BF16, BF16, BF16, "tokens", False),
    (300, 1, 1, 40, 0, False, "qk", F32, BF16, BF16, "tokens", False),
]


def rope_reference(x, w, cos, sin, eps, interleaved):
    """[tokens, heads, d] f64: the values, and a bound on the size of the terms behind each."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2: r])
    c, s = cos.double()[:, None], sin.double()[:, None]
    y, size = x.clone(), x.abs()
    for part, v, m in (((slice(0, r, 2) if interleaved else slice(0, r // 2)), a * c - b * s, (a * c).abs() + (b * s).abs()),
                       ((slice(1, r, 2) if interleaved else slice(r // 2, r)), b * c + a * s, (b * c).abs() + (a * s).abs())):
        y[..., part], size[..., part] = v, m
    return y, size


def near(got, want, size, dtype):
    # f32 arithmetic: up to 8 roundings and the mean over up to 256 squares before the one to the output's type
    tol = size * 2.0 ** -19 + U[dtype] * want.abs() * 1.01 + (2.0 ** -25 if dtype == F16 else 1e-30)
    return bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("i", range(len(ROPE)))
def test_rope(attention, i):
    t, hq, hk, d, rot, inter, norms, it, ot, ct, layout, joined = ROPE[i]
    g = _gen(400 + i)
    page = 16
    k_cache, v_cache, _ = make_cache(g, [t + 40], page, hk, d, ct, layout)
    k_cache.copy_(_randn(g, *k_cache.shape, dtype=ct))
    v_cache.copy_(_randn(g, *v_cache.shape, dtype=ct))
    rows = _randn(g, t, (hq + 2 * hk) * d, dtype=it) * 2
    q, k, v = rows.split([hq * d, hk * d, hk * d], 1)
    q, k, v = (x.view(t, -1, d) if joined else x.reshape(t, -1, d).clone() for x in (q, k, v))
    cos, sin = attention.rope_tables(5000, rot) if rot else (torch.empty(5000, 0, device="cuda"),) * 2
    pos = torch.randint(0, 5000, (t,), generator=g, device="cuda").to(torch.int32)
    slots = torch.randperm(k_cache.shape[0] * page, generator=g, device="cuda")[:t].contiguous()
    slots[t // 2:: 7] = -1
    qw, kw = ((1 + 0.3 * _randn(g, d)) if n in norms else None for n in "qk")
    before = k_cache.clone(), v_cache.clone()
    got = attention.rope_append(q, k, v, pos, cos, sin, k_cache, v_cache, slots, qw, kw, 1e-5, inter, out_dtype=ot)
    ops.check_device_status()
    assert got.dtype == ot and got.is_contiguous()
    c, s = cos[pos.long()], sin[pos.long()]
    assert near(got, *rope_reference(q, qw, c, s, 1e-5, inter), ot)
    kept = slots >= 0
    at = slots[kept] // page, slots[kept] % page
    want, size = rope_reference(k, kw, c, s, 1e-5, inter)
    assert near(k_cache[at], want[kept], size[kept], ct)
    assert torch.equal(v_cache[at], v[kept].to(ct))
    for cache, old in zip((k_cache, v_cache), before):
        cache[at] = old[at]
        assert torch.equal(cache, old), "a place that no slot names was written"


def test_rope_in_place_and_unaligned(attention):
    g = _gen(13)
    t, hq, hk, d = 30, 8, 2, 64
    k_cache, v_cache = attention.new_cache(8, 16, hk, d)
    cos, sin = attention.rope_tables(100, d)
    pos, slots = torch.arange(t, device="cuda", dtype=torch.int32), torch.arange(t, device="cuda")
    q, k, v = (_randn(g, t, h, d, dtype=BF16) for h in (hq, hk, hk))
    want = attention.rope_append(q, k, v, pos, cos, sin, k_cache, v_cache, slots)
    kept = k_cache.clone()
    odd = _randn(g, t, hq, d + 3, dtype=BF16)
    odd[..., 1:d + 1] = q
    k_cache.zero_()
    assert torch.equal(attention.rope_append(odd[..., 1:d + 1], k, v, pos, cos, sin, k_cache, v_cache, slots), want)
    assert torch.equal(k_cache, kept)
    assert attention.rope_append(q, k, v, pos, cos, sin, k_cache, v_cache, slots, out=q) is q and torch.equal(q, want)


def test_rope_bad_positions_and_slots(attention):
    g = _gen(14)
    k_cache, v_cache = attention.new_cache(4, 16, 2, 64)
    cos, sin = attention.rope_tables(10, 64)
    q, k, v = (_randn(g, 2, h, 64) for h in (4, 2, 2))
    for pos, slots in (([0, 10], [0, 1]), ([0, -1], [0, 1]), ([0, 1], [0, 64])):
        k_cache.zero_()
        out = attention.rope_append(q, k, v, _ints(pos), cos, sin, k_cache, v_cache, _ints(slots, torch.int64))
        with pytest.raises(_cabi.B200QError, match="out of range"):
            ops.check_device_status()
        assert torch.equal(out[0], q[0]) and k_cache.view(64, 2, 64)[0].any() and not k_cache.view(64, 2, 64)[1:].any()


def test_rope_refusals(attention):
    k_cache, v_cache = attention.new_cache(4, 16, 2, 64)
    cos, sin = attention.rope_tables(10, 64)
    q, k, v = (torch.zeros(3, h, 64, device="cuda") for h in (4, 2, 2))
    fine = [q, k, v, _ints([0, 1, 2]), cos, sin, k_cache, v_cache, _ints([0, 1, 2], torch.int64)]
    attention.rope_append(*fine)
    for at, value, text in [(0, q.bfloat16(), "alike"), (0, q.double(), "F32, BF16 or F16"), (1, k[:2], "key-value heads"), (2, v[..., :32], "key-value heads"),
                            (3, fine[3].long(), "positions"), (8, fine[8].int(), "slots"), (4, cos.double(), "cos and sin"), (5, sin[:5], "cos and sin"),
                            (4, torch.zeros(10, 40, device="cuda"), "cos and sin"), (6, k_cache.float(), "BF16 or F16"), (0, q.cpu(), "CUDA device")]:
        args = list(fine)
        args[at] = value
        with pytest.raises(QuantError, match=text):
            attention.rope_append(*args)
    with pytest.raises(QuantError, match="q_weight"):
        attention.rope_append(*fine, q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(QuantError, match="out must be"):
        attention.rope_append(*fine, out=torch.empty(3, 4, 32, device="cuda"))
    with pytest.raises(QuantError, match="output must be"):
        attention.rope_append(*fine, out_dtype=torch.float64)


# ------------------------------------------------------------------------------- compiled entry points and the Python form


def _outcome(call):
    try:
        r = call()
    except Exception as e:
        return type(e), str(e)
    return [t.clone() for t in (r if isinstance(r, tuple) else (r,))]


def test_both_forms_agree(attention, monkeypatch):
    """The compiled entry points and the Python form: the same bits, the same refusals in the same words."""
    from boostr_b200 import tensor

    assert tensor.hostops().__name__ == "boostr_b200._hostops", "the compiled entry points are not built"
    q, k, v, t, n = _fine(attention)
    cu = _ints([0, 1, 2])
    cos, sin = attention.rope_tables(40, 64)
    kr, vr, pos, slots = q[:, :2], q[:, 2:], _ints([3, 4]), _ints([0, 17], torch.int64)
    kc, vc = attention.new_cache(4, 16, 2, 64)
    w = torch.rand(64, device="cuda")
    out = torch.zeros_like(q)
    wide = torch.cat([q, q], 2)[..., 32:96]
    ws = attention.decode_workspace(4, 2, 64)
    calls = {}
    for name, f in (("decode", attention.paged_decode), ("prompt", lambda q, *a, **o: attention.paged_prompt(q, cu, *a, **o))):
        c = lambda *a, f=f, **o: lambda: f(*a, **o)  # noqa: E731
        calls.update({
            f"{name}": c(q, k, v, t, n), f"{name} lse": c(q, k, v, t, n, return_lse=True), f"{name} f32 out": c(q, k, v, t, n, out_dtype=F32),
            f"{name} out": c(q, k, v, t, n, out=out), f"{name} scale": c(q, k, v, t, n, scale=0.2, window=9, sinks=2), f"{name} int scale": c(q, k, v, t, n, scale=1),
            f"{name} strided": c(wide, k, v, t, n), f"{name} f32": c(q.float(), k, v, t, n), f"{name} half": c(q.half(), k, v, t, n),
            f"{name} lens": c(q, k, v, t, n[:1]), f"{name} long": c(q, k, v, t, n.long()), f"{name} window": c(q, k, v, t, n, window=-2),
            f"{name} f64": c(q, k, v, t, n, out_dtype=torch.float64), f"{name} out shape": c(q, k, v, t, n, out=out[:1]),
            f"{name} heads": c(q[:, :3], k, v, t, n), f"{name} empty": c(q[:0], k, v, t[:0], n[:0]) if name == "decode" else c(q[:0], k, v, t, n),
        })
    calls["decode workspace"] = lambda: attention.paged_decode(q, k, v, t, n, workspace=ws)
    calls["decode small workspace"] = lambda: attention.paged_decode(q, k, v, t, n, workspace=ws[:4096])
    calls["decode host workspace"] = lambda: attention.paged_decode(q, k, v, t, n, workspace=ws.cpu())
    rope = lambda *a, **o: lambda: (attention.rope_append(*a, **o), kc.clone(), vc.clone())  # noqa: E731
    calls.update({
        "rope": rope(q, kr, vr, pos, cos, sin, kc, vc, slots), "rope norm": rope(q, kr, vr, pos, cos, sin, kc, vc, slots, w, w, 1),
        "rope inter": rope(q, kr, vr, pos, cos, sin, kc, vc, slots, None, w, interleaved=True, out_dtype=F32),
        "rope out": rope(q, kr, vr, pos, cos, sin, kc, vc, slots, out=torch.zeros_like(q)), "rope type": rope(q, kr.float(), vr, pos, cos, sin, kc, vc, slots),
        "rope slots": rope(q, kr, vr, pos, cos, sin, kc, vc, slots.int()), "rope weight": rope(q, kr, vr, pos, cos, sin, kc, vc, slots, w[:32]),
        "rope f64": rope(q, kr, vr, pos, cos, sin, kc, vc, slots, out_dtype=torch.float64), "rope table": rope(q, kr, vr, pos, cos[:3], sin, kc, vc, slots),
    })
    table = lambda: _ints([[7, -1], [8, -1]])  # noqa: E731
    sl = lambda *a: lambda: tuple(attention.paged_slots(*a))  # noqa: E731
    calls.update({"slots": sl(_ints([3, 16]), _ints([14, 2]), table(), 16, _ints([1, 2, 3]), _ints([3]), 18),
                  "slots padded": sl(_ints([3, 16]), _ints([14, 2]), table(), 16, _ints([1, 2, 3]), _ints([1]), 20),
                  "slots none": sl(_ints([3, 16]), _ints([0, 0]), table(), 16, _ints([1]), _ints([1]), 0),
                  "slots page": sl(_ints([3, 16]), _ints([0, 0]), table(), 0, _ints([1]), _ints([1]), 0),
                  "slots tokens": sl(_ints([3, 16]), _ints([0, 0]), table(), 16, _ints([1]), _ints([1]), -1),
                  "slots lens": sl(_ints([3, 16]), _ints([0]), table(), 16, _ints([1]), _ints([1]), 1)})
    compiled = {}
    for name, call in calls.items():
        kc.zero_(), vc.zero_()
        compiled[name] = _outcome(call)
    monkeypatch.setattr(tensor, "_hostops", tensor._PythonForms)
    for name, call in calls.items():
        kc.zero_(), vc.zero_()
        a, b = compiled[name], _outcome(call)
        assert type(a) is type(b), (name, a, b)
        if isinstance(a, tuple):
            assert a == b, name
        else:
            assert len(a) == len(b) and all(x.shape == y.shape and x.dtype == y.dtype and torch.equal(x, y) for x, y in zip(a, b)), name
    refused = {n for n, r in compiled.items() if isinstance(r, tuple)}
    assert refused == {x for x in calls if x.split(" ", 1)[-1] in ("half", "lens", "long", "window", "f64", "out shape", "heads", "small workspace", "host workspace",
                                                                    "type", "slots", "weight", "table", "page", "tokens")} - {"slots"} | {"prompt f32"}, refused
    ops.check_device_status()


def test_scratch_of_threads_and_streams(attention):
    """Threads on one stream and on their own: the joins of one call do not meet another's."""
    import threading

    g = _gen(15)
    sets = []
    for lens in ([9000], [700, 20000], [64] * 30):
        k, v, t = make_cache(g, lens, 16, 2, 128, BF16)
        q = _randn(g, len(lens), 16, 128, dtype=BF16)
        sets.append((q, k, v, t, _ints(lens)))
    want = [attention.paged_decode(*s) for s in sets]
    torch.cuda.synchronize()
    shared, errors = torch.cuda.Stream(), []

    def work(i):
        try:
            with torch.cuda.stream(shared if i < 3 else torch.cuda.Stream()):
                for r in range(40):
                    j = (i + r) % len(sets)
                    if not torch.equal(attention.paged_decode(*sets[j]), want[j]):
                        raise AssertionError(f"thread {i}, pass {r}")
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    ops.check_device_status()
