"""The kernels of the 8-bit path against their definition in 64 bits (``int8_refs``), at the sizes, masks and values where they
can go wrong, and what they refuse.

Tolerances. 2^-24 is half a unit of a 32-bit value. A code is held to the value it stands for: half a step, and what the
value may be off before it is rounded, times up to 127 steps. Products are exact sums, scaled with three roundings."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

import int8_refs as ref
from tinyserve_b200.engine.arena import Arena
from tinyserve_b200.kernels import ops

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
U = 2.0 ** -24


def rnd(*shape, dtype=torch.float32, seed=0, scale=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)


def rows_hold(codes, scales, y, off) -> None:
    """``codes * scales`` stand for ``y`` (64 bits), each of which the kernel may have had ``off`` (relative) from it."""
    width = y.shape[1]
    want = ref.scale_of(ref.most_of(y))
    assert torch.equal(torch.isnan(scales), torch.isnan(want))
    fine = torch.isfinite(want)
    assert bool(((scales.double() - want).abs()[fine] <= (off + 2 * U) * want[fine]).all())
    assert not codes[:, width:].any() and not codes[~fine].any()
    values = codes[fine, :width].double() * scales[fine].double()[:, None]
    assert bool(((values - y[fine]).abs() <= want[fine][:, None] * (0.5 + 127 * (2 * off + 6 * U)) + 1e-300).all())
    assert int(codes.to(torch.int32).abs().max()) <= 127


# ------------------------------------------------------------------------------------------------ rows
WIDTHS = [1, 7, 16, 72, 200, 1000, 1024, 2048, 4096, 4100, 5120, 8192, 12288, 16384, 20000]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("t", [1, 5, 333])
def test_norm_rows(dtype, width, t) -> None:
    """A sum of squares of h values in 32 bits in any order: (h + 2) U at most, half of that in its root; four roundings more."""
    resid, delta = rnd(t, width, seed=1, scale=3.0), rnd(t, width, dtype=dtype, seed=2)
    weight = (1 + rnd(width, seed=3, scale=0.1)).to(dtype)
    for d in (delta, None):
        for out_width in {width, ops.int8_width(width)}:
            x, codes = resid.clone(), torch.full((t, out_width), 99, dtype=torch.int8, device="cuda")
            scales = torch.full((t,), math.nan, device="cuda")
            ops.add_rms_norm_int8(x, d, weight, 1e-5, codes, scales)
            want = resid if d is None else resid + d.float()
            assert torch.equal(x, want)
            rows_hold(codes, scales, ref.normed(want, weight, 1e-5), (width / 2 + 6) * U)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", "none"])
@pytest.mark.parametrize("t", [1, 6, 333])
def test_activated_rows(dtype, width, activation, t) -> None:
    """silu: the exponential to 2 units, a sum, a division, a product: 8 U. gelu: the tanh to 2 units of a value next to -1 is
    2 U absolutely, and gate (1 + tanh) is small there: an error of |gate up| U in place of a relative one."""
    x = rnd(t, width * (1 if activation == "none" else 2), dtype=dtype, seed=4, scale=2.0)
    for out_width in {width, ops.int8_width(width)}:
        codes = torch.full((t, out_width), 99, dtype=torch.int8, device="cuda")
        scales = torch.full((t,), math.nan, device="cuda")
        ops.act_mul_int8(x, codes, scales, activation)
        y = ref.activated(x, activation)
        if activation == "gelu_tanh":
            g, u = x.double().chunk(2, 1)
            loose = float((g * u).abs().amax() * 4 * U)
            fine = scales.double() * 127 > 0
            assert bool(fine.all())
            values = codes[:, :width].double() * scales.double()[:, None]
            assert bool(((values - y).abs() <= scales.double()[:, None] * (0.5 + 127 * 24 * U) + loose).all())
            assert bool(((scales.double() * 127 - y.abs().amax(1)).abs() <= 24 * U * y.abs().amax(1) + loose).all())
            assert not codes[:, width:].any()
        else:
            rows_hold(codes, scales, y, 8 * U)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [40, 1024, 4096, 4100, 20000])
def test_rows_of_nothing_and_of_no_numbers(dtype, width) -> None:
    """Zeros, values too small for a scale, the largest values, infinities and NaNs at either end of a row: only their own row sees them."""
    x = rnd(9, width, dtype=dtype, seed=5)
    x[1] = 0
    x[2] = 2.0 ** -105
    x[3] *= 2.0 ** 120 / float(x[3].abs().max())
    x[4, 0] = math.inf
    x[5, -1] = -math.inf
    x[6, width // 2] = math.nan
    x[7] *= 2.0 ** -90
    codes, scales = torch.full((9, width), 99, dtype=torch.int8, device="cuda"), torch.full((9,), 99.0, device="cuda")
    ops.act_mul_int8(x, codes, scales, "none")
    assert torch.isnan(scales).tolist() == [False] * 4 + [True] * 3 + [False] * 2
    assert scales[1] == 0 and scales[2] == 0 and not codes[1:3].any() and not codes[4:7].any()
    rows_hold(codes[[0, 3, 7, 8]], scales[[0, 3, 7, 8]], x[[0, 3, 7, 8]].double(), 2 * U)
    # the norm: a NaN in the stream, in the pending output; a stream of zeros is normed to zeros
    resid = rnd(4, width, seed=6)
    resid[1, 3] = math.nan
    resid[3] = 0
    delta = torch.zeros(4, width, dtype=dtype, device="cuda")
    delta[2, -1] = math.inf
    out, s = torch.empty(4, width, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    ops.add_rms_norm_int8(resid, delta, torch.ones(width, dtype=dtype, device="cuda"), 1e-5, out, s)
    assert torch.isnan(s).tolist() == [False, True, True, False] and s[3] == 0 and not out[1:].any()


@gpu
def test_rows_on_a_stream_of_their_own() -> None:
    """The launch goes to the current stream, behind what is queued there."""
    side = torch.cuda.Stream()
    x = rnd(700, 2 * 4096, dtype=torch.bfloat16, seed=7)
    codes, scales = torch.empty(700, 4096, dtype=torch.int8, device="cuda"), torch.empty(700, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = torch.zeros_like(x)
        for _ in range(20):
            y = y + x / 20
        ops.act_mul_int8(y, codes, scales)
        got = codes.clone(), scales.clone()
    side.synchronize()
    want = torch.empty_like(codes), torch.empty_like(scales)
    ops.act_mul_int8(y, *want)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_values(dtype) -> None:
    codes = torch.randint(-127, 128, (7, 3, 5, 24), dtype=torch.int8, device="cuda")
    scales = rnd(7, 3, seed=8).abs()
    rows = torch.tensor([6, 0, 6, 3], dtype=torch.int32, device="cuda")
    out, want = (torch.empty(4, 3, 5, 24, dtype=dtype, device="cuda") for _ in range(2))
    ops.int8_values(codes, scales, out, rows=rows)
    want.copy_((codes.float() * scales[..., None, None])[rows.long()])
    assert torch.equal(out, want)
    for width, padded in ((16, 16), (1000, 1008), (4096, 4096), (37, 48)):
        codes, scales = torch.randint(-127, 128, (33, padded), dtype=torch.int8, device="cuda"), rnd(33, seed=9)
        out = torch.empty(33, width, dtype=dtype, device="cuda")
        ops.int8_values(codes, scales, out)
        assert torch.equal(out, (codes.float() * scales[:, None]).to(dtype)[:, :width])
    outside = torch.tensor([-1, 2, 33], dtype=torch.int32, device="cuda")
    out = torch.empty(3, 37, dtype=dtype, device="cuda")
    ops.int8_values(codes, scales, out, rows=outside)
    assert torch.isnan(out).all(1).tolist() == [True, False, True]


# ------------------------------------------------------------------------------------------------ the product
def product_holds(x, xs, w, ws, out) -> None:
    want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()[None, :]
    step = 4 * U if out.dtype == torch.float32 else 2.0 ** -8 + 4 * U
    assert bool(((out.double() - want).abs() <= step * want.abs()).all())


def product_inputs(m, n, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-127, 128, (m, k), dtype=torch.int8, generator=g, device="cuda")
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, generator=g, device="cuda")
    return x, torch.rand(m, generator=g, device="cuda") + 0.1, w, torch.rand(n, generator=g, device="cuda") + 0.1


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [16, 48, 128, 144, 1040, 4096])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 33), (1, 1000), (2, 128), (7, 129), (8, 4096), (16, 256), (17, 100), (33, 512), (64, 2048), (65, 127),
                                 (100, 640), (128, 1024), (129, 255), (200, 2056), (257, 300), (300, 4096), (513, 1537), (1100, 2304)])
def test_product(dtype, m, n, k) -> None:
    x, xs, w, ws = product_inputs(m, n, k, seed=m + n + k)
    out = torch.full((m, n), math.nan, dtype=dtype, device="cuda")
    ops.gemm_int8(x, xs, w, ws, out)
    product_holds(x, xs, w, ws, out)


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 24576, 4096), (3, 5000, 12288), (16, 6144, 1024), (37, 6144, 4096), (130, 8192, 512), (2048, 4096, 1024),
                                   (999, 24576, 256), (5, 151936, 1024)])
def test_product_of_larger_matrices(m, n, k) -> None:
    x, xs, w, ws = product_inputs(m, n, k, seed=3)
    for dtype in DTYPES:
        out = torch.full((m, n), math.nan, dtype=dtype, device="cuda")
        ops.gemm_int8(x, xs, w, ws, out)
        product_holds(x, xs, w, ws, out)


@gpu
@pytest.mark.parametrize("m", [1, 20, 150, 600])
def test_product_at_the_ends_of_the_integers(m) -> None:
    """The deepest product of the largest codes, either sign, lies inside 32 bits; -128, which the rows above never hold, counts as itself."""
    k = ops.INT8_MAX_DEPTH
    x = torch.full((m, k), 127, dtype=torch.int8, device="cuda")
    w = torch.full((130, k), 127, dtype=torch.int8, device="cuda")
    w[1::2] = -127
    ones = torch.ones(m, device="cuda"), torch.ones(130, device="cuda")
    out = torch.empty(m, 130, device="cuda")
    ops.gemm_int8(x, ones[0], w, ones[1], out)
    assert bool((out.double().abs() == float(torch.tensor(127 * 127 * k, dtype=torch.float32))).all())
    assert bool((out[:, 0::2] > 0).all()) and bool((out[:, 1::2] < 0).all())
    x = torch.full((m, 64), -128, dtype=torch.int8, device="cuda")
    w = torch.full((130, 64), -128, dtype=torch.int8, device="cuda")
    ops.gemm_int8(x, ones[0], w, ones[1], out)
    assert bool((out == 64 * 128 * 128).all())


@gpu
@pytest.mark.parametrize("m", [4, 40, 300])
def test_product_of_rows_without_numbers(m) -> None:
    x, xs, w, ws = product_inputs(m, 200, 256)
    xs[2], xs[3], ws[7] = math.nan, 0.0, math.nan
    out = torch.empty(m, 200, dtype=torch.bfloat16, device="cuda")
    ops.gemm_int8(x, xs, w, ws, out)
    bad = torch.isnan(out)
    assert bool(bad[2].all()) and bool(bad[:, 7].all()) and int(bad.sum()) == m + 200 - 1
    assert bool((out[3][~bad[3]] == 0).all())


@gpu
def test_a_product_follows_the_rows_it_reads() -> None:
    """The row kernel and the product queued one behind the other, many times over other rows: none reads the rows before."""
    w, ws = ops.int8_weight(rnd(2048, 1024, dtype=torch.bfloat16, seed=1, scale=0.02))
    codes, scales = torch.empty(24, 1024, dtype=torch.int8, device="cuda"), torch.empty(24, device="cuda")
    xs = [rnd(24, 1024, dtype=torch.bfloat16, seed=10 + i, scale=float(i + 1)) for i in range(12)]
    outs = [torch.empty(24, 2048, device="cuda") for _ in xs]
    for x, out in zip(xs, outs):
        ops.act_mul_int8(x, codes, scales, "none")
        ops.gemm_int8(codes, scales, w, ws, out)
    for x, out in zip(xs, outs):
        c, s = torch.empty_like(codes), torch.empty_like(scales)
        ops.act_mul_int8(x, c, s, "none")
        torch.cuda.synchronize()
        product_holds(c, s, w, ws, out)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_8_bit_weight(dtype) -> None:
    w = rnd(70, 100, dtype=dtype, seed=2)
    codes, scales = ops.int8_weight(w)
    assert codes.shape == (70, 112)
    rows_hold(codes, scales, w.double(), 2 * U)


# ------------------------------------------------------------------------------------------------ the cache
def step_of(query_lens, context_lens, dtype=torch.bfloat16):
    """A step of these requests: new tokens and all tokens of each."""
    i32 = dict(dtype=torch.int32, device="cuda")
    b = len(query_lens)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(query_lens).cumsum(0)])
    return SimpleNamespace(
        num_tokens=sum(query_lens), num_seqs=b, query_lens=list(query_lens), context_lens=list(context_lens), cu_query_lens=cu.to(**i32),
        context_lens_dev=torch.tensor(context_lens, **i32), decode_seqs=torch.tensor([i for i in range(b) if query_lens[i] == 1], **i32),
        prefill_seqs=torch.tensor([i for i in range(b) if query_lens[i] > 1], **i32), num_decode=sum(n == 1 for n in query_lens),
        num_prefill=sum(n > 1 for n in query_lens), max_query_len=max(query_lens), max_context_len=max(context_lens), recorded=False,
        prompt_heads=None, dtype=dtype, arena=Arena("cuda"))


def tables_for(context_lens, page, spare=3, seed=0):
    used = [-(-n // page) for n in context_lens]
    order = torch.randperm(sum(used) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tables = torch.full((len(used), max(max(used), 1)), 2 ** 30, dtype=torch.int32)      # entries that nothing may follow
    at = 0
    for r, n in enumerate(used):
        tables[r, :n] = order[at: at + n]
        at += n
    return tables.cuda(), sum(used) + spare


def cache_of(pages, hkv, page, d, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = [torch.randint(-127, 128, (pages, hkv, page, d), dtype=torch.int8, generator=g, device="cuda") for _ in range(2)]
    return [*codes, *(torch.rand(pages, hkv, generator=g, device="cuda") * 0.01 + 0.005 for _ in range(2))]


def write_holds(k, v, before, after, page, tables, ctx) -> None:
    want = [x.clone() for x in before]
    unrounded = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in want[:2]]
    ref.kv_write_int8(k, v, *want, page, tables, ctx, unrounded=unrounded)
    for n in (0, 1):
        codes, scales, to_codes, to_scales = after[n], after[n + 2], want[n], want[n + 2]
        assert torch.equal(torch.isnan(scales), torch.isnan(to_scales))
        fine = torch.isfinite(to_scales)
        assert bool(((scales - to_scales).abs()[fine] <= 2 * U * to_scales[fine]).all())
        # a code may fall to either side where its value (up to 127, six roundings) lies next to the middle between two
        apart = (codes.int() - to_codes.int()).abs()
        middle = (unrounded[n] - unrounded[n].floor() - 0.5).abs() <= 127 * 6 * U
        assert int(apart.max()) <= 1 and not bool((apart.bool() & ~middle).any())
        values = codes.double() * scales.double()[..., None, None]
        exact = to_codes.double() * to_scales.double()[..., None, None]
        assert bool(((values - exact).abs() <= (apart + 127 * 4 * U) * to_scales.double()[..., None, None])[fine].all())
        same = torch.ones(codes.shape[:3], dtype=torch.bool, device="cuda")
        quiet = torch.ones(scales.shape[0], dtype=torch.bool, device="cuda")
        for r, block, lo, hi, _ in ref.touched(ctx, page):
            p = int(tables[r, block])
            quiet[p] = False
            same[p, :, : hi - block * page] = False
        assert torch.equal(codes[same], before[n][same]), "codes of other pages, or behind the last token"
        assert torch.equal(scales[quiet], before[n + 2][quiet])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", [(1, 16, 1), (2, 64, 16), (8, 128, 16), (3, 80, 24), (2, 256, 8), (5, 36, 16), (2, 128, 64), (1, 128, 256)])
@pytest.mark.parametrize("query_lens,context_lens", [([1], [1]), ([1, 1, 1, 1], [16, 17, 40, 300]), ([37], [37]), ([5, 1, 100, 33], [5, 64, 205, 50]),
                                                     ([1] * 40, list(range(1, 41)))])
def test_cache_write(dtype, hkv, d, page, query_lens, context_lens) -> None:
    ctx = step_of(query_lens, context_lens, dtype)
    tables, pages = tables_for(context_lens, page)
    cache = cache_of(pages, hkv, page, d)
    k, v = rnd(ctx.num_tokens, hkv, d, dtype=dtype, seed=1), rnd(ctx.num_tokens, hkv, d, dtype=dtype, seed=2, scale=0.3)
    before = [x.clone() for x in cache]
    ops.kv_write_int8(k, v, *cache, page, tables, ctx)
    write_holds(k, v, before, cache, page, tables, ctx)


@gpu
def test_a_page_filled_token_by_token() -> None:
    """Louder and louder tokens: each rounds the page again, by half a step of the scale of that moment at most; then a quiet
    one, which changes nothing that is there."""
    page, d = 16, 64
    tables, pages = tables_for([16], page)
    cache = cache_of(pages, 1, page, d)
    rows = rnd(16, 1, d, seed=3) * torch.linspace(0.2, 2.0, 16, device="cuda")[:, None, None]
    rows[15] *= 0.01
    budget = torch.zeros((), dtype=torch.float64, device="cuda")
    p = int(tables[0, 0])
    for n in range(1, 17):
        was = [x.clone() for x in cache]
        ops.kv_write_int8(rows[n - 1: n], rows[n - 1: n], *cache, page, tables, step_of([1], [n]))
        scale = cache[2][p, 0].double()
        budget = budget + (0.5 + 1e-4) * scale if n == 1 or cache[2][p, 0] != was[2][p, 0] else torch.maximum(budget, (0.5 + 1e-4) * scale)
        off = (cache[0][p, 0, :n].double() * scale - rows[:n, 0].double()).abs().max()
        assert off <= budget
    assert torch.equal(cache[0][p, 0, :15], was[0][p, 0, :15]) and torch.equal(cache[2], was[2])


@gpu
@pytest.mark.parametrize("where", ["new", "held", "tiny"])
def test_a_page_without_numbers(where) -> None:
    page, d, hkv = 16, 64, 3
    tables, pages = tables_for([20], page)
    cache = cache_of(pages, hkv, page, d)
    rows = rnd(1, hkv, d, seed=4)
    p = int(tables[0, 1])
    if where == "new":
        rows[0, 1, 5] = math.inf
    elif where == "held":
        cache[2][p, 1], cache[3][p, 1] = math.nan, math.nan
    else:
        rows[:] = 2.0 ** -110
        cache[2][p], cache[3][p] = 0.0, 0.0
    before = [x.clone() for x in cache]
    ops.kv_write_int8(rows, rows, *cache, page, tables, step_of([1], [20]))
    if where == "tiny":
        assert not cache[2][p].any() and not cache[0][p, :, 3].any()
        return
    assert torch.isnan(cache[2][p]).tolist() == [False, True, False] and not cache[0][p, 1, :4].any()
    write_holds(rows, rows, before, cache, page, tables, step_of([1], [20]))


# ------------------------------------------------------------------------------------------------ attention
def attention_holds(q, cache, page, tables, ctx, window, out, scale) -> None:
    """32 bits: sums of D products and of n terms. bf16: the weights, and where the pages are read as bf16 the keys and
    values, are rounded to 8 bits (2^-9 each; the keys' moves a score by 2^-9 of sum |q k| at most, a weight and its sum by twice
    that), and the result is (2^-9, of a value that may be off)."""
    want, size, reach = ref.attended(q, *cache, page, tables, ctx, scale, window)
    got = out.view(q.shape).double()
    n = ctx.max_context_len
    if q.dtype == torch.float32:
        bound = size * (2 * (q.shape[2] + 8) * U * reach + (n + 32) * U)
    else:
        bound = size * (3 * 2.0 ** -9 + 2 * 2.0 ** -9 * reach) + 2.0 ** -8 * want.abs()
    assert bool(((got - want).abs() <= bound + 1e-30).all()), float(((got - want).abs() - bound).max())


def quiet_elsewhere(cache, tables, context_lens, page, query_lens, window):
    """NaN scales on every page that no query of the step may look at."""
    seen = torch.zeros(cache[0].shape[0], dtype=torch.bool)
    for r, n in enumerate(context_lens):
        lo = max(0, n - query_lens[r] - window + 1) if window else 0
        for b in range(lo // page, -(-n // page)):
            seen[int(tables[r, b])] = True
        if window:
            tables[r, : lo // page] = 2 ** 30
    for s in cache[2:]:
        s[~seen] = math.nan


LAYOUTS = [(16, 8, 128, 16), (32, 8, 128, 16), (4, 4, 64, 16), (8, 1, 64, 32), (16, 1, 128, 8), (40, 2, 128, 16), (6, 2, 80, 16), (4, 2, 256, 24), (3, 1, 36, 5),
           (4, 2, 128, 64), (12, 2, 96, 16)]


def attend(q, cache, page, tables, ctx, window, scale):
    out = torch.full((q.shape[0], q.shape[1] * q.shape[2]), math.nan, dtype=q.dtype, device="cuda")
    ops.paged_attention_int8(q, *cache, page, tables, ctx, scale, window, out)
    return out


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", LAYOUTS)
@pytest.mark.parametrize("window", [0, 1, 20, 500])
def test_attention_of_single_tokens(dtype, hq, hkv, d, page, window) -> None:
    for lens in ([1], [1, 2, 15, 16, 17, 64, 129, 700], [2500], [33] * 70):
        ctx = step_of([1] * len(lens), lens, dtype)
        tables, pages = tables_for(lens, page)
        cache = cache_of(pages, hkv, page, d)
        quiet_elsewhere(cache, tables, lens, page, [1] * len(lens), window)
        q = rnd(len(lens), hq, d, dtype=dtype, seed=5)
        out = attend(q, cache, page, tables, ctx, window, d ** -0.5)
        attention_holds(q, cache, page, tables, ctx, window, out, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", LAYOUTS)
@pytest.mark.parametrize("window", [0, 20])
def test_attention_of_portions(dtype, hq, hkv, d, page, window) -> None:
    """Prompts and portions of them beside single tokens, in one step; two tokens, a few, many."""
    for new, lens in (([2], [2]), ([3, 1, 5, 1], [3, 90, 40, 1]), ([130], [130]), ([70, 1, 200], [300, 44, 200])):
        ctx = step_of(new, lens, dtype)
        tables, pages = tables_for(lens, page)
        cache = cache_of(pages, hkv, page, d)
        quiet_elsewhere(cache, tables, lens, page, new, window)
        q = rnd(sum(new), hq, d, dtype=dtype, seed=6)
        out = attend(q, cache, page, tables, ctx, window, d ** -0.5)
        attention_holds(q, cache, page, tables, ctx, window, out, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 4, 40])
def test_attention_where_one_key_takes_all(dtype, new) -> None:
    """Scores of hundreds: all weight on the best key, the running maximum moves late or never; and scores all equal (queries of
    zeros)."""
    hq, hkv, d, page, n = 8, 2, 128, 16, 1000
    tables, pages = tables_for([n], page)
    cache = cache_of(pages, hkv, page, d)
    ctx = step_of([new], [n], dtype)
    for scale, late in ((20.0, False), (20.0, True), (0.0, False)):
        q = rnd(new, hq, d, dtype=dtype, seed=7) if scale else torch.zeros(new, hq, d, dtype=dtype, device="cuda")
        scale = scale or 1.0
        if late:
            cache[2][int(tables[0, (n - new) // page])] *= 8          # the last page that every query sees is the loudest
        out = attend(q, cache, page, tables, ctx, 0, scale)
        want = ref.attended(q, *cache, page, tables, ctx, scale, 0)[0]
        assert torch.isfinite(out).all()
        if q.any():       # rounding moves scores of thousands by more than 1: the best key's value comes out where it is far ahead
            k = (cache[0][tables[0].long()].double() * cache[2][tables[0].long()].double()[..., None, None]).transpose(0, 1).reshape(hkv, -1, d)
            s = torch.einsum("ihd,hjd->ihj", q.double(), k.repeat_interleave(hq // hkv, 0)) * scale
            s = s.masked_fill(torch.arange(k.shape[1], device="cuda")[None, None] > (n - new + torch.arange(new, device="cuda"))[:, None, None], -math.inf)
            top = s.topk(2, -1).values
            slack = 40 + 2.0 ** -8 * (s.masked_fill(s == -math.inf, 0).abs().amax(-1) * 12)
            clear = (top[..., 0] - top[..., 1]) > slack
            assert bool(((out.view(q.shape).double() - want).abs()[clear] <= 2.0 ** -7 * want.abs()[clear] + 1e-6).all())
        else:
            attention_holds(q, cache, page, tables, ctx, 0, out, scale)


@gpu
def test_attention_after_writes() -> None:
    """A prompt in portions, then tokens one by one, through the write and the attention, against attention over the rows
    themselves: what 8 bits lose of a key or value is half a step, a few times over where a page's scale grew."""
    hq, hkv, d, page, total = 8, 2, 64, 16, 150
    rows = [rnd(total, hkv, d, seed=s) for s in (1, 2)]
    q = rnd(total, hq, d, seed=3)
    tables, pages = tables_for([total], page)
    cache = cache_of(pages, hkv, page, d)
    outs, at = [], 0
    for new in [70, 1, 1, 33, 2] + [1] * (total - 107):
        ctx = step_of([new], [at + new], torch.float32)
        ops.kv_write_int8(rows[0][at: at + new], rows[1][at: at + new], *cache, page, tables, ctx)
        outs.append(attend(q[at: at + new], cache, page, tables, ctx, 0, d ** -0.5))
        at += new
    k, v = (x.double().repeat_interleave(hq // hkv, 1) for x in rows)
    s = torch.einsum("ihd,jhd->hij", q.double(), k) * d ** -0.5
    p = torch.softmax(s.masked_fill(torch.ones(total, total, device="cuda").triu(1).bool(), -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", p, v)
    off = (torch.cat(outs).view(total, hq, d).double() - want).norm() / want.norm()
    assert off < 0.02          # a step is 1/127 of 3 to 4 deviations: an error of 0.9 % of one deviation a value, keys and values


# ------------------------------------------------------------------------------------------------ refusals
def refuses(match, f, *args, **kw) -> None:
    with pytest.raises(ops.KernelError, match=match):
        f(*args, **kw)


def test_what_rows_and_products_refuse() -> None:
    e = lambda *s, dtype=torch.int8: torch.empty(*s, dtype=dtype)      # noqa: E731
    f = lambda *s: torch.empty(*s)                                      # noqa: E731
    refuses("out must be", ops.act_mul_int8, f(3, 40), e(3, 21), f(3), "none")
    refuses("out must be", ops.act_mul_int8, f(3, 40), e(3, 64), f(3), "none")
    refuses("one scale", ops.act_mul_int8, f(3, 40), e(3, 48), f(4), "none")
    refuses("two equal halves", ops.act_mul_int8, f(3, 41), e(3, 32), f(3))
    refuses("unknown activation", ops.act_mul_int8, f(3, 40), e(3, 20), f(3), "relu")
    refuses("shape", ops.add_rms_norm_int8, f(3, 40), f(3, 41), f(40), 1e-5, e(3, 40), f(3))
    refuses("shape", ops.add_rms_norm_int8, f(3, 40), None, f(41), 1e-5, e(3, 40), f(3))
    refuses("multiple of 16", ops.gemm_int8, e(2, 40), f(2), e(5, 40), f(5), f(2, 5))
    refuses("multiple of 16", ops.gemm_int8, e(1, 131088), f(1), e(1, 131088), f(1), f(1, 1))
    refuses("shape", ops.gemm_int8, e(2, 48), f(2), e(5, 32), f(5), f(2, 5))
    refuses("shape", ops.gemm_int8, e(2, 48), f(3), e(5, 48), f(5), f(2, 5))
    refuses("CUDA tensor", ops.gemm_int8, e(2, 48), f(2), e(5, 48), f(5), f(2, 5))
    refuses("first one or two", ops.int8_values, e(3, 4, 5), f(4), f(3, 4, 5))
    refuses("codes' shape", ops.int8_values, e(3, 16), f(3), f(3, 17))
    refuses("codes' shape", ops.int8_values, e(3, 2, 16), f(3, 2), f(3, 2, 8))


def test_what_the_cache_refuses() -> None:
    e = lambda *s: torch.empty(*s, dtype=torch.int8)                    # noqa: E731
    f = lambda *s: torch.empty(*s)                                      # noqa: E731
    ctx = SimpleNamespace(num_tokens=3, num_seqs=2)
    tables = torch.zeros(2, 4, dtype=torch.int32)
    good = (e(9, 2, 16, 64), e(9, 2, 16, 64), f(9, 2), f(9, 2), 16, tables, ctx)
    k = f(3, 2, 64)
    refuses("alike", ops.kv_write_int8, k, f(3, 2, 32), *good)
    refuses("alike", ops.kv_write_int8, f(4, 2, 64), f(4, 2, 64), *good)
    refuses("layout", ops.kv_write_int8, k, k, good[0], e(9, 2, 8, 64), *good[2:])
    refuses("scales", ops.kv_write_int8, k, k, *good[:3], f(9, 3), *good[4:])
    refuses("block_tables", ops.kv_write_int8, k, k, *good[:5], tables[:1], ctx)
    refuses("CUDA tensor", ops.kv_write_int8, k, k, *good[:6], SimpleNamespace(num_tokens=3, num_seqs=2, max_query_len=2))
    refuses("head grouping", ops.paged_attention_int8, f(3, 5, 64), *good, 1.0, 0, f(3, 320))
    refuses("scale", ops.paged_attention_int8, f(3, 4, 64), *good, 0.0, 0, f(3, 256))
    refuses("window", ops.paged_attention_int8, f(3, 4, 64), *good, 1.0, -1, f(3, 256))
    big = (e(9, 2, 16, 512), e(9, 2, 16, 512), *good[2:])
    refuses("head size", ops.paged_attention_int8, f(3, 4, 512), *big, 1.0, 0, f(3, 2048))


def test_attention_refuses_rows_that_are_not_the_steps() -> None:
    """The kernels find a request's rows by the step's lengths: fewer rows than the step has tokens would be read behind their end."""
    ctx = SimpleNamespace(num_tokens=3, num_seqs=2, max_query_len=2, num_prefill=1, num_decode=1, max_context_len=40)
    cache = (*(torch.empty(9, 2, 16, 64, dtype=torch.int8) for _ in range(2)), torch.empty(9, 2), torch.empty(9, 2))
    tables = torch.zeros(2, 4, dtype=torch.int32)
    for t in (0, 2, 4):
        refuses("row per token", ops.paged_attention_int8, torch.empty(t, 4, 64), *cache, 16, tables, ctx, 1.0, 0, torch.empty(t, 256))


@gpu
def test_what_the_kernels_refuse_of_tensors() -> None:
    """Types, layouts and addresses that only a tensor on the device shows."""
    x, xs, w, ws = product_inputs(4, 32, 64)
    out = torch.empty(4, 32, device="cuda")
    refuses("contiguous", ops.gemm_int8, product_inputs(4, 32, 128)[0][:, :64], xs, w, ws, out)
    refuses("int8", ops.gemm_int8, x.to(torch.uint8), xs, w, ws, out)
    refuses("float32", ops.gemm_int8, x, xs.double(), w, ws, out)
    refuses("dtype", ops.gemm_int8, x, xs, w, ws, out.half())
    store = torch.empty(4 * 64 + 16, dtype=torch.int8, device="cuda")
    refuses("not supported", ops.gemm_int8, store[1: 257].view(4, 64), xs, w, ws, out)
    refuses("dtype", ops.act_mul_int8, torch.empty(4, 64, device="cuda", dtype=torch.float16), x, xs, "none")


@gpu
def test_nothing_to_do() -> None:
    z = dict(device="cuda")
    ops.act_mul_int8(torch.empty(0, 64, **z), torch.empty(0, 32, dtype=torch.int8, **z), torch.empty(0, **z))
    ops.add_rms_norm_int8(torch.empty(0, 64, **z), None, torch.empty(64, **z), 1e-5, torch.empty(0, 64, dtype=torch.int8, **z), torch.empty(0, **z))
    ops.gemm_int8(torch.empty(0, 64, dtype=torch.int8, **z), torch.empty(0, **z), torch.empty(8, 64, dtype=torch.int8, **z), torch.empty(8, **z),
                  torch.empty(0, 8, **z))
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (4, 4, 64, 16), (16, 1, 128, 8), (12, 2, 96, 32), (6, 2, 80, 16)])
@pytest.mark.parametrize("window", [0, 20])
def test_attention_of_many_requests(hq, hkv, d, page, window) -> None:
    """More requests than run at once, lengths of one, far apart, all alike (the longest are begun first), and a step in which
    not all requests bring one token."""
    for lens in ([3000] + [9] * 80 + [2500, 2500], [1] * 400, list(range(1, 129)), list(range(1, 300)), [70] * 90):
        ctx = step_of([1] * len(lens), lens)
        tables, pages = tables_for(lens, page)
        cache = cache_of(pages, hkv, page, d)
        quiet_elsewhere(cache, tables, lens, page, [1] * len(lens), window)
        q = rnd(len(lens), hq, d, dtype=torch.bfloat16, seed=5)
        out = attend(q, cache, page, tables, ctx, window, d ** -0.5)
        attention_holds(q, cache, page, tables, ctx, window, out, d ** -0.5)
    new, lens = [1, 3, 1, 40] * 30, [90, 50, 1, 300] * 30
    ctx = step_of(new, lens)
    tables, pages = tables_for(lens, page)
    cache = cache_of(pages, hkv, page, d)
    quiet_elsewhere(cache, tables, lens, page, new, window)
    q = rnd(sum(new), hq, d, dtype=torch.bfloat16, seed=6)
    attention_holds(q, cache, page, tables, ctx, window, attend(q, cache, page, tables, ctx, window, d ** -0.5), d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("copies", [1, 40])
def test_requests_without_keys_get_zeros(dtype, copies) -> None:
    """A length of zero, in front, between and behind."""
    lens = [0, 40, 0, 0, 300, 0] * copies
    ctx = step_of([1] * len(lens), lens, dtype)
    tables, pages = tables_for(lens, 16)
    cache = cache_of(pages, 2, 16, 128)
    q = rnd(len(lens), 8, 128, dtype=dtype, seed=5)
    out = attend(q, cache, 16, tables, ctx, 0, 0.1)
    some = [i for i, n in enumerate(lens) if n]
    assert not out[[i for i, n in enumerate(lens) if not n]].any()
    attention_holds(q[some], cache, 16, tables[some], step_of([1] * len(some), [lens[i] for i in some], dtype), 0, out[some].contiguous(), 0.1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [40, 1024, 4096, 20000])
def test_norm_of_small_rows(dtype, width) -> None:
    """A stream whose products with the weight have no reciprocal in 32 bits but whose norm has: between 2^-126 and 2^-100."""
    resid = rnd(4, width, seed=8) * torch.tensor([1e-31, 3e-33, 1.0, 1e-30], device="cuda")[:, None]
    weight = (1 + rnd(width, seed=3, scale=0.1)).to(dtype)
    codes, scales = torch.full((4, width), 99, dtype=torch.int8, device="cuda"), torch.full((4,), math.nan, device="cuda")
    ops.add_rms_norm_int8(resid.clone(), None, weight, 1e-6, codes, scales)
    assert bool((scales > 0).all())
    rows_hold(codes, scales, ref.normed(resid, weight, 1e-6), (width / 2 + 6) * U)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (6, 2, 80, 16), (4, 2, 96, 32), (4, 2, 64, 8), (3, 1, 36, 5)])
@pytest.mark.parametrize("new", [3, 30, 700])
@pytest.mark.parametrize("window", [0, 40])
def test_pages_without_numbers_reach_the_rows_that_see_them(dtype, hq, hkv, d, page, new, window) -> None:
    """A page whose keys or whose values are no numbers makes NaN of the queries that see it, and of them alone: earlier ones and
    those whose window has passed it are as if it held anything else."""
    n = 50 * page * max(1, 700 // (40 * page)) + 1                 # the last token begins a page
    ctx = step_of([new], [n], dtype)
    tables, pages = tables_for([n], page)
    q = rnd(new, hq, d, dtype=dtype, seed=6)
    first = n - new
    blocks = {(n - 1) // page, (n - 1) // page - 1, (max(0, first - window + 1) if window else first) // page}
    at = torch.arange(first, n, device="cuda")
    for block in sorted(blocks):
        for which in (2, 3):
            cache = cache_of(pages, hkv, page, d)
            head = (block + which) % hkv
            numbers = [x.clone() for x in cache]
            cache[which][int(tables[0, block]), head] = math.nan
            out = attend(q, cache, page, tables, ctx, window, d ** -0.5).view(new, hkv, hq // hkv, d)
            sees = (at >= block * page) & ((at - window < (block + 1) * page - 1) if window else (at >= 0))
            assert torch.equal(torch.isnan(out[:, head]).all(-1).all(-1), sees) and torch.equal(torch.isnan(out[:, head]).any(-1).any(-1), sees)
            blind = out.clone()
            blind[sees, head] = 0
            want, size, reach = ref.attended(q, *numbers, page, tables, ctx, d ** -0.5, window)
            want.view(new, hkv, hq // hkv, d)[sees, head] = 0
            if dtype == torch.float32:
                bound = size * (2 * (d + 8) * U * reach + (n + 32) * U)
            else:
                bound = size * (3 * 2.0 ** -9 + 2 * 2.0 ** -9 * reach) + 2.0 ** -8 * want.abs()
            assert bool(((blind.view(new, hq, d).double() - want).abs() <= bound + 1e-30).all())


@gpu
@pytest.mark.parametrize("m,n,k", [(37, 512, 1024), (100, 4096, 4096), (600, 8192, 1024)])
def test_a_wait_of_the_product_that_runs_out(m, n, k) -> None:
    """Copies that never come end as an error on the host; the next launch is right again."""
    from test_wait_failure_gpu import error_code, lost_copies

    assert (ops.int8_product_form(m, n, k)[0] == 256) == (m == 600)
    x, xs, w, ws = product_inputs(m, n, k)
    out = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    with lost_copies():
        ops.gemm_int8(x, xs, w, ws, out)
        assert error_code() == 1
        with pytest.raises(ops.KernelError, match="gemm_tcgen05"):
            ops.check_device_errors()
    ops.gemm_int8(x, xs, w, ws, out)
    ops.check_device_errors()
    product_holds(x, xs, w, ws, out)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 16, 17, 64, 100, 128, 300])
@pytest.mark.parametrize("n,k", [(1000, 144), (777, 1040), (2050, 2048), (96, 4096)])
def test_product_in_every_form(dtype, m, n, k, monkeypatch) -> None:
    """Tiles of every height, with slices where they are taken, whatever the rule would choose for the shape."""
    rows = 16 if m <= 16 else 32 if m <= 32 else 64 if m <= 64 else 128
    x, xs, w, ws = product_inputs(m, n, k)
    for form in ((rows, 1, 8), (rows, 1, 96), (rows, 1, 128), (rows, 1, 136), (rows, 1, 200), (rows, 1, 256), (rows, 2, 64), (rows, 2, 128), (256, 1, 256)):
        monkeypatch.setattr(ops, "int8_product_form", lambda *_: form)
        out = torch.full((m, n), math.nan, dtype=dtype, device="cuda")
        ops.gemm_int8(x, xs, w, ws, out)
        product_holds(x, xs, w, ws, out)
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("m,n,k", [(12, 20000, 1024), (64, 24576, 512), (128, 37888, 272), (40, 37889, 128), (100, 80000, 144), (64, 9472, 1024), (65, 9472, 2048),
                                   (33, 2048, 1024), (20, 5000, 768)])
def test_product_where_the_form_changes(m, n, k) -> None:
    x, xs, w, ws = product_inputs(m, n, k)
    out = torch.full((m, n), math.nan, dtype=torch.bfloat16, device="cuda")
    ops.gemm_int8(x, xs, w, ws, out)
    product_holds(x, xs, w, ws, out)
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [32, 64, 192, 320, 520])
@pytest.mark.parametrize("k", [16, 256])
def test_product_of_more_rows_than_one_turn_of_tiles(dtype, n, k) -> None:
    """More than 74 tiles of 256 rows: a pair of CTAs takes several tiles of the last columns one after the other, each with an odd
    number of pieces of the result (of 32 or 64 columns) among these widths. Every element, several times over."""
    m = 3 * 74 * 256 + 77
    assert ops.int8_product_form(m, n, k)[0] == 256
    x, xs, w, ws = product_inputs(m, n, k, seed=n + k)
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    for _ in range(3):
        out.fill_(math.nan)
        ops.gemm_int8(x, xs, w, ws, out)
        product_holds(x, xs, w, ws, out)
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [16, 20, 37, 300, 301])
def test_values_of_no_items_at_all(dtype, width) -> None:
    """Every item asked for lies outside: NaN, in each of the readers' forms (vectors of 16 and 4, single codes, long groups)."""
    rows = torch.tensor([0, -1, 5], dtype=torch.int32, device="cuda")
    out = torch.zeros(3, width, dtype=dtype, device="cuda")
    ops.int8_values(torch.empty(0, width, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"), out, rows=rows)
    assert bool(torch.isnan(out).all())
    out = torch.zeros(3, 2, 5, width, dtype=dtype, device="cuda")
    ops.int8_values(torch.empty(0, 2, 5, width, dtype=torch.int8, device="cuda"), torch.empty(0, 2, device="cuda"), out, rows=rows)
    assert bool(torch.isnan(out).all())


def portions_case(new, lens, hq, hkv, d, page, dtype, window=0, seed=0):
    ctx = step_of(new, lens, dtype)
    tables, pages = tables_for(lens, page)
    cache = cache_of(pages, hkv, page, d, seed=seed)
    quiet_elsewhere(cache, tables, lens, page, new, window)
    return ctx, tables, cache, rnd(sum(new), hq, d, dtype=dtype, seed=6)


@gpu
def test_portions_take_no_more_scratch_than_they_may() -> None:
    """Pages of all requests of the step, as values, would be 1.3 GB here; a second layer works in the memory of the first."""
    ctx, tables, cache, q = portions_case([32, 1] * 40, [8192, 9] * 40, 32, 8, 128, 16, torch.bfloat16)
    for _ in range(2):
        ctx.arena.next_frame()
        out = attend(q, cache, 16, tables, ctx, 0, 0.09)
    assert ctx.arena.reserved_bytes <= (512 << 20) + (1 << 20)
    attention_holds(q, cache, 16, tables, ctx, 0, out, 0.09)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (4, 4, 64, 16), (6, 2, 80, 16), (12, 2, 96, 32), (3, 1, 36, 5), (4, 2, 256, 24)])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("pages_at_once", [0, 20, 60, 100])
def test_portions_with_little_scratch(dtype, hq, hkv, d, page, window, pages_at_once, monkeypatch) -> None:
    """Some requests at a time, beside single tokens between them; requests that alone are beyond the scratch go over the codes."""
    new = [200, 1, 31, 2, 1, 300, 90, 1, 64]
    lens = [20 * page, 30, 33 * page - 1 if page > 1 else 40, 2, 700, 59 * page, 19 * page, 1, 90 * page]
    new = [min(a, b) for a, b in zip(new, lens)]
    ctx, tables, cache, q = portions_case(new, lens, hq, hkv, d, page, dtype, window)
    monkeypatch.setattr(ops, "_int8_direct_rows", lambda *_: 0)
    limit = pages_at_once * 2 * hkv * page * d * q.element_size()
    monkeypatch.setattr(ops, "INT8_PORTIONS_SCRATCH_BYTES", limit)
    out = attend(q, cache, page, tables, ctx, window, d ** -0.5)
    attention_holds(q, cache, page, tables, ctx, window, out, d ** -0.5)
    assert (ctx.arena.reserved_bytes > 0) == (pages_at_once > 0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_portions_without_memory_for_scratch(dtype, monkeypatch) -> None:
    """They go over the codes; the arena is as it was."""
    new, lens = [100, 1, 300], [1000, 40, 2000]
    ctx, tables, cache, q = portions_case(new, lens, 8, 2, 128, 16, dtype)
    monkeypatch.setattr(ops, "_int8_direct_rows", lambda *_: 0)
    lost = []

    def take(self, nbytes):
        lost.append(nbytes)
        raise torch.cuda.OutOfMemoryError("no memory")

    monkeypatch.setattr(Arena, "take_for_call", take)
    out = attend(q, cache, 16, tables, ctx, 0, 0.09)
    assert len(lost) == 1 and lost[0] >= 3000 * 2 * 2 * 128 * q.element_size()
    attention_holds(q, cache, 16, tables, ctx, 0, out, 0.09)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (4, 4, 64, 8), (12, 2, 96, 16), (6, 2, 80, 16), (3, 1, 36, 5)])
@pytest.mark.parametrize("new,n", [(1, 1), (1, 300), (1, 3000), (5, 90), (7, 7)])
def test_attention_where_every_score_is_far_below_zero(dtype, hq, hkv, d, page, new, n) -> None:
    """Scores of -1e32, far enough apart that the best key takes all: its values come out, as for any other scores. Head by head
    all keys' elements are of one sign and the queries of the other; a key's codes are its place, so the first one scores best."""
    ctx = step_of([new], [n], dtype)
    tables, pages = tables_for([n], page)
    cache = cache_of(pages, hkv, page, d)
    cache[0][:] = 0
    cache[2][:] = 1.0
    place = torch.arange(n, device="cuda")
    cache[0][tables[0].long()[place // page], :, place % page] = torch.clamp(place + 1, max=127).to(torch.int8)[:, None, None]
    q = torch.full((new, hq, d), -1e30, dtype=dtype, device="cuda")
    out = attend(q, cache, page, tables, ctx, 0, 1.0).view(new, hkv, hq // hkv, d)
    first = (cache[1][int(tables[0, 0]), :, 0].double() * cache[3][int(tables[0, 0])].double()[:, None])[None, :, None]
    step = 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -7
    assert bool(((out.double() - first).abs() <= step * first.abs()).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", [(8, 128, 16), (5, 36, 16), (3, 50, 7)])
def test_codes_of_the_cache_are_quotients_rounded_once(dtype, hkv, d, page) -> None:
    """A value over its scale, correctly rounded, to the nearest code: many bf16 values lie half a step between two (half of the
    largest is 63.5 steps), where one rounding more falls to the other side. The same for what a page held, in its new scale."""
    new, lens = [90 * page] + [1] * 60, [90 * page] + [page + 3] * 60
    ctx = step_of(new, lens, dtype)
    tables, pages = tables_for(lens, page)
    cache = cache_of(pages, hkv, page, d)
    k, v = rnd(ctx.num_tokens, hkv, d, dtype=dtype, seed=1), rnd(ctx.num_tokens, hkv, d, dtype=dtype, seed=2, scale=0.3)
    before = [x.clone() for x in cache]
    ops.kv_write_int8(k, v, *cache, page, tables, ctx)
    seen = 0
    for rows, codes, scales, had, had_scale in ((k, cache[0], cache[2], before[0], before[2]), (v, cache[1], cache[3], before[1], before[3])):
        for r, block, lo, hi, shift in ref.touched(ctx, page):
            p, held = int(tables[r, block]), lo - block * page
            s = scales[p][:, None, None]
            fresh = rows[lo + shift: hi + shift].float().transpose(0, 1)
            assert torch.equal(codes[p, :, held: held + hi - lo], torch.round(fresh / s).to(torch.int8))
            kept, grew = had[p, :, :held], (scales[p] > had_scale[p])[:, None, None]
            again = torch.round(kept.float() * had_scale[p][:, None, None] / s).to(torch.int8)
            assert torch.equal(codes[p, :, :held], torch.where(grew, again, kept))
            seen += int(grew.sum()) if held else 0
    assert seen > 20


@gpu
def test_portions_some_at_a_time_with_indices_checked(monkeypatch) -> None:
    """The check of block tables (``TINYSERVE_B200_CHECK_INDICES``) looks at all rows of the table of values, of which a run of
    requests fills its own: the others hold pages that are there, whatever the memory held before."""
    new, lens = [200, 1, 100, 300], [320, 30, 640, 944]
    ctx, tables, cache, q = portions_case(new, lens, 8, 2, 128, 16, torch.bfloat16)
    tables[tables >= cache[0].shape[0]] = 0
    ctx.arena.take((1 << 20,), torch.int32).fill_(2 ** 30)
    ctx.arena.begin_step()
    monkeypatch.setattr(ops, "CHECK_INDICES", True)
    monkeypatch.setattr(ops, "_int8_direct_rows", lambda *_: 0)
    monkeypatch.setattr(ops, "INT8_PORTIONS_SCRATCH_BYTES", 60 * 2 * 2 * 16 * 128 * 2)
    out = attend(q, cache, 16, tables, ctx, 0, 0.09)
    attention_holds(q, cache, 16, tables, ctx, 0, out, 0.09)
