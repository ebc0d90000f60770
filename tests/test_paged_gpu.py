"""The paged KV cache operators against plain implementations in 64 bits.

Attention bounds, per output element, derived from the arithmetic: with A =
sum_j w_j |v_j| (w the softmax weights, sink included in their sum) and u the
unit roundoff of the tensors' type (2^-8 bf16, 2^-11 f16),
  16-bit types: the weights are rounded to the type once (u A), the result
    once (u |out|), fp32 sums and exponentials add less than 2^-14 A; a f16
    weight below the normal range keeps an absolute error, under 2^-14 A too.
    A f16 result below its normal range is 2^-25 off at least (half the
    spacing of f16 there), whoever computes it.
  fp32: a score's error is that of a D-term sum, about 2^-24 sqrt(D) S with S
    = scale sum_i |q_i k_i|, and it scales the weight; sums over n keys add
    2^-24 sqrt(n), the exponential and its argument (up to 2 S) a few units.
    The factor 4 covers the tail of these random sums.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _torch():
    import torch
    return torch


def _dt(name):
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


_handle = []


def handle():
    if not _handle:
        from picchio_b200 import Attention
        _handle.append(Attention())
    return _handle[0]


def reference(q, k, v, p0, sinks, window, scale, dtype):
    """One request: q [n, H, D] at positions p0 ..., k and v [L, KH, D].  The
    outputs and the bound on their error, in 64 bits."""
    torch = _torch()
    n, H, D = q.shape
    L, KH = k.shape[0], k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    pos = torch.arange(p0, p0 + n, device=q.device)[:, None]
    key = torch.arange(L, device=q.device)[None]
    sees = key <= pos
    if window:
        sees &= key > pos - window
    for h in range(H):
        kk, vv = k[:, h // (H // KH)].double(), v[:, h // (H // KH)].double()
        qq = q[:, h].double()
        used = sees.any(0)  # what no row sees may hold anything
        kk = torch.where(used[:, None], kk, 0.0)
        s = torch.where(sees, qq @ kk.T * scale, -math.inf)
        top = s.amax(1, keepdim=True) if L else torch.full((n, 1), -math.inf, dtype=torch.float64, device=q.device)
        if sinks is not None:
            top = top.clamp(min=float(sinks[h]))
        top = torch.where(top == -math.inf, 0.0, top)
        w = torch.exp(s - top)
        tot = w.sum(1, keepdim=True) + (torch.exp(float(sinks[h]) - top) if sinks is not None else 0.0)
        w = w / torch.where(tot == 0, 1.0, tot)
        # an unseen key has no part, whatever V holds: finite V in one product, the rest row by row
        fin = torch.where(torch.isfinite(vv), vv, 0.0)
        o, A = w @ fin, w @ fin.abs()
        for j in (~torch.isfinite(vv)).any(1).nonzero().flatten().tolist():
            bad = torch.where(torch.isfinite(vv[j]), 0.0, vv[j])
            o = torch.where(sees[:, j, None], o + bad, o)
        out[:, h] = o
        if dtype == "f32":
            S = torch.where(sees, qq.abs() @ kk.abs().T * scale, 0.0).amax(1, keepdim=True) if L else tot * 0
            bound[:, h] = 2.0 ** -24 * (4 * math.sqrt(D) * S + 4 * math.sqrt(max(L, 1)) + 4 * S + 16) * A
        else:
            bound[:, h] = U[dtype] * (o.abs() + A) + 2.0 ** -14 * A + (2.0 ** -25 if dtype == "f16" else 0.0)
    return out, bound * 1.02 + 1e-30


def close(got, want, bound):
    torch = _torch()
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & ~inf, torch.zeros_like(inf)) and torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    over = ((got - want).abs() / bound)[ok]
    assert over.numel() == 0 or float(over.max()) <= 1.0, float(over.max())


def gen(seed):
    torch = _torch()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_paged(reqs, page, H, KH, D, dtype, seed, spare=3, heads_first=False, garbage=True, q_gap=8):
    """Requests (positions in all, new ones): a cache whose unused rows hold
    NaN, tables whose unused entries are -1, q as a slice of wider rows."""
    torch = _torch()
    g, dt = gen(seed), _dt(dtype)
    total, new = [r[0] for r in reqs], [r[1] for r in reqs]
    have = [-(-t // page) for t in total]
    n_pages = sum(have) + spare
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    shape = (n_pages, KH, page, D) if heads_first else (n_pages, page, KH, D)
    kp = torch.randn(shape, generator=g, device="cuda").to(dt)
    vp = torch.randn(shape, generator=g, device="cuda").to(dt)
    if heads_first:
        kp, vp = kp.permute(0, 2, 1, 3), vp.permute(0, 2, 1, 3)
    table = torch.full((len(reqs), max(max(have), 1) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = order[at:at + h]
        at += h
    if garbage:
        live = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
        for b, t in enumerate(total):
            for j in range(have[b]):
                live[int(table[b, j]), :max(0, min(page, t - j * page))] = True
        kp[~live] = float("nan")
        vp[~live] = float("nan")
    T = sum(new)
    rows = torch.randn(T + 2, H * D + q_gap, generator=g, device="cuda").to(dt)
    q = (rows * 1.5)[:T, :H * D].view(T, H, D) if q_gap else (rows * 1.5)[:T].view(T, H, D)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    kv = torch.tensor(total, dtype=torch.int32, device="cuda")
    return q, kp, vp, table, cu, kv


def gathered(pages, table, b, n):
    page = pages.shape[1]
    if n == 0:
        return pages[:0].flatten(0, 1)
    return pages[table[b, :-(-n // page)].long()].flatten(0, 1)[:n]


def check_paged(reqs, page, H, KH, D, dtype, sinks, window, seed=1, scale=None, **kw):
    torch = _torch()
    q, kp, vp, table, cu, kv = make_paged(reqs, page, H, KH, D, dtype, seed, **kw)
    sk = torch.randn(H, generator=gen(seed + 1), device="cuda") if sinks else None
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    got = handle().paged(q, kp, vp, table, cu, kv, sinks=sk, window=window, scale=scale, out=out)
    handle().check()
    assert got is out
    for b, (total, new) in enumerate(reqs):
        r = slice(int(cu[b]), int(cu[b + 1]))
        want, bound = reference(q[r], gathered(kp, table, b, total), gathered(vp, table, b, total), total - new, sk,
                                window, D ** -0.5 if scale is None else scale, dtype)
        close(out[r], want, bound)


DTYPES = ["f32", "f16", "bf16"]
# (positions, new ones): one token at first, ends of pages and tiles, no new rows, long ones
DECODE = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (64, 1), (65, 1), (127, 1), (128, 1), (129, 1), (700, 1), (5, 0),
          (0, 0), (1500, 1)]
CHUNKS = [(40, 40), (1, 1), (300, 37), (0, 0), (513, 130), (129, 2), (64, 64), (1000, 17), (257, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KH,D,page", [(64, 8, 64, 16), (8, 8, 128, 32), (10, 2, 80, 8), (7, 1, 40, 24)])
@pytest.mark.parametrize("window", [0, 128, 3])
def test_paged_single_tokens(dtype, H, KH, D, page, window):
    check_paged(DECODE, page, H, KH, D, dtype, True, window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KH,D,page", [(16, 2, 64, 16), (8, 8, 128, 64), (6, 2, 96, 40), (48, 1, 8, 8)])
@pytest.mark.parametrize("window", [0, 128, 1])
def test_paged_chunks(dtype, H, KH, D, page, window):
    check_paged(CHUNKS, page, H, KH, D, dtype, window != 0, window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_long_rows_are_split(dtype):
    """One token, and a few, over long contexts: several blocks share a row."""
    check_paged([(9001, 1)], 16, 64, 8, 64, dtype, True, 0)
    check_paged([(9001, 3), (20, 1)], 32, 8, 4, 128, dtype, False, 0)
    check_paged([(6000, 70)], 16, 16, 2, 64, dtype, True, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32)])
def test_paged_many_tiles_a_block(dtype, D, page):
    """Each block goes through its ring of tiles many times, and from item to
    item, with warps ahead of one another."""
    check_paged([(2900 + 37 * (i % 11), 1) for i in range(48)], page, 32, 4, D, dtype, True, 0)
    check_paged([(2500 + 91 * (i % 7), 1 + 60 * (i % 4 == 3)) for i in range(24)], page, 32, 8, D, dtype, False, 700)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_rows_without_keys_give_zeros(dtype):
    """Fewer positions in the cache than new rows: the first rows stand before
    position 0 and see nothing, with and without sinks."""
    for sinks in (False, True):
        check_paged([(0, 3), (2, 5), (40, 100), (0, 1), (130, 400)], 16, 8, 2, 64, dtype, sinks, 0)
        check_paged([(0, 3), (2, 5), (40, 100), (0, 1), (130, 400)], 16, 8, 2, 64, dtype, sinks, 16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_windows_beyond_every_position(dtype):
    """Windows up to the type's largest and past it: all keys, also for rows
    before position 0."""
    for window in (1 << 30, 2**31 - 1, 1 << 40):
        check_paged([(0, 3), (40, 100), (0, 1), (130, 400), (300, 1), (77, 5)], 16, 8, 2, 64, dtype, False, window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_many_requests(dtype):
    reqs = [(1 + (37 * i) % 90, 1 + i % 2) for i in range(700)]
    check_paged([(max(t, n), n) for t, n in reqs], 8, 4, 1, 32, dtype, True, 0)
    check_paged([(60 + i % 5, 20 + i % 17) for i in range(400)], 16, 4, 2, 64, dtype, False, 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_cache_of_other_strides(dtype):
    """Pages laid out heads first, q without a gap, a scale of its own."""
    check_paged(CHUNKS, 16, 16, 2, 64, dtype, True, 0, heads_first=True, q_gap=0, scale=0.2)
    check_paged(DECODE, 16, 16, 2, 64, dtype, True, 0, heads_first=True, q_gap=0, scale=0.2)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("new", [1, 90])
def test_paged_cache_beyond_32_bit_offsets(dtype, new):
    """Pages more than 2^31 elements into the cache."""
    torch = _torch()
    D, page, n_pages = 64, 64, 530000
    if dtype == "f32":
        D = 32
        n_pages *= 2
    kp = torch.empty(n_pages, page, 1, D, dtype=_dt(dtype), device="cuda")
    vp = torch.empty(n_pages, page, 1, D, dtype=_dt(dtype), device="cuda")
    total = 200
    pages = [n_pages - 1, 0, n_pages - 3, n_pages // 2]
    table = torch.tensor([pages], dtype=torch.int32, device="cuda")
    g = gen(3)
    for p in pages:
        kp[p] = torch.randn(page, 1, D, generator=g, device="cuda").to(kp.dtype)
        vp[p] = torch.randn(page, 1, D, generator=g, device="cuda").to(kp.dtype)
    q = torch.randn(new, 4, D, generator=g, device="cuda").to(kp.dtype)
    cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    kv = torch.tensor([total], dtype=torch.int32, device="cuda")
    out = handle().paged(q, kp, vp, table, cu, kv)
    want, bound = reference(q, gathered(kp, table, 0, total), gathered(vp, table, 0, total), total - new, None, 0,
                            D ** -0.5, dtype)
    close(out, want, bound)
    # the store reaches the same slots
    from picchio_b200 import kv_store
    k = torch.randn(2, 1, D, generator=g, device="cuda").to(kp.dtype)
    slots = torch.tensor([(n_pages - 1) * page + 5, 3], dtype=torch.int64, device="cuda")
    kv_store(kp, vp, k, k * 2, slots)
    assert torch.equal(kp[n_pages - 1, 5], k[0]) and torch.equal(vp[0, 3], k[1] * 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[1], [5, 1, 130], [0, 64, 0, 65], [300, 17, 513], [1100]])
@pytest.mark.parametrize("H,KH,D,window,sinks", [(64, 8, 64, 0, True), (64, 8, 64, 128, True), (6, 2, 128, 0, False),
                                                 (5, 1, 72, 7, True), (4, 4, 16, 0, False)])
def test_packed(dtype, lens, H, KH, D, window, sinks):
    torch = _torch()
    T = sum(lens)
    rows = (torch.randn(T, (H + 2 * KH) * D + 8, generator=gen(T + H), device="cuda") * 1.3).to(_dt(dtype))
    q = rows[:, :H * D].view(T, H, D)
    k = rows[:, H * D:(H + KH) * D].view(T, KH, D)
    v = rows[:, (H + KH) * D:(H + 2 * KH) * D].view(T, KH, D)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    sk = torch.randn(H, generator=gen(9), device="cuda") if sinks else None
    out = handle().packed(q, k, v, cu, sinks=sk, window=window)
    handle().check()
    for b in range(len(lens)):
        r = slice(int(cu[b]), int(cu[b + 1]))
        want, bound = reference(q[r], k[r], v[r], 0, sk, window, D ** -0.5, dtype)
        close(out[r], want, bound)


def best_time(f):
    """The least of 12 times of 8 calls."""
    torch = _torch()
    times = []
    for _ in range(12):
        e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        e[0].record()
        for _ in range(8):
            f()
        e[1].record()
        e[1].synchronize()
        times.append(e[0].elapsed_time(e[1]))
    return min(times)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_empty_prompts_cost_little(dtype):
    """A thread block's way over slots without a prompt is short (one by one
    the 511 behind the last prompt took as long as the prompt)."""
    torch = _torch()
    n = 1000
    q, k, v = (torch.randn(n, h, 64, generator=gen(5), device="cuda").to(_dt(dtype)) for h in (64, 8, 8))
    alone = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    among = torch.tensor([0] * 513 + [n] * 512, dtype=torch.int32, device="cuda")
    gaps = torch.tensor([0] * 300 + [n // 3] * 300 + [n // 2] * 31 + [n] * 394, dtype=torch.int32, device="cuda")
    assert torch.equal(handle().packed(q, k, v, among), handle().packed(q, k, v, alone))
    out = handle().packed(q, k, v, gaps)
    for a, b in ((0, n // 3), (n // 3, n // 2), (n // 2, n)):
        want, bound = reference(q[a:b], k[a:b], v[a:b], 0, None, 0, 0.125, dtype)
        close(out[a:b], want, bound)
    one, many = best_time(lambda: handle().packed(q, k, v, alone)), best_time(lambda: handle().packed(q, k, v, among))
    assert many < 1.6 * one, (many, one)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KH,D", [(8, 2, 64), (8, 1, 64), (8, 2, 128), (40, 1, 64), (96, 1, 8)])
@pytest.mark.parametrize("window", [0, 100])
def test_paged_one_long_among_many(dtype, H, KH, D, window):
    """One chunk among slots without a request, and beside single tokens: the
    longest request has far more rows than the average."""
    check_paged([(0, 0)] * 20 + [(500, 170)] + [(0, 0)] * 40, 16, H, KH, D, dtype, True, window)
    check_paged([(50, 1)] * 9 + [(300, 90)] + [(0, 0)] * 40 + [(20, 1)] * 9, 16, H, KH, D, dtype, False, window)
    check_paged([(300, 1), (0, 0), (260, 6), (0, 0)], 16, H, KH, D, dtype, False, window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_idle_slots_cost_little(dtype):
    """A prompt among slots without a request runs as it does alone (a choice of
    the kernel by the average rows a request made it 4 times as long in 16 bits,
    twice in fp32)."""
    alone, among = (make_paged(r, 16, 64, 8, 64, dtype, 3, garbage=False)
                    for r in ([(1500, 1500)], [(0, 0)] * 512 + [(1500, 1500)] + [(0, 0)] * 511))
    one, many = best_time(lambda: handle().paged(*alone)), best_time(lambda: handle().paged(*among))
    assert many < 1.6 * one, (many, one)


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_rows_are_left_alone(dtype):
    """Rows past the last request's are not written, whatever q holds there."""
    torch = _torch()
    for new in (1, 60):
        q, kp, vp, table, cu, kv = make_paged([(70, new), (200, new)], 16, 8, 2, 64, dtype, 6)
        rows = torch.full((2 * new + 150, 8, 64), float("nan"), dtype=q.dtype, device="cuda")
        rows[:2 * new] = q
        out = torch.full_like(rows, 7.0)
        handle().paged(rows, kp, vp, table, cu, kv, out=out)
        assert torch.isfinite(out[:2 * new].float()).all() and (out[2 * new:] == 7.0).all()
        out.fill_(7.0)
        k, v = (torch.randn(2 * new + 150, 2, 64, device="cuda").to(q.dtype) for _ in range(2))
        k[2 * new:] = v[2 * new:] = float("nan")
        handle().packed(rows, k, v, cu, out=out)
        assert torch.isfinite(out[:2 * new].float()).all() and (out[2 * new:] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads_that_are_one(dtype):
    """K and V expanded over heads (strides of zero): no tensor map has them."""
    torch = _torch()
    n, H, KH, D = 333, 6, 3, 64
    g = gen(31)
    q = torch.randn(n, H, D, generator=g, device="cuda").to(_dt(dtype))
    k, v = (torch.randn(n, 1, D, generator=g, device="cuda").to(_dt(dtype)).expand(n, KH, D) for _ in range(2))
    cu = torch.tensor([0, 100, n], dtype=torch.int32, device="cuda")
    out = handle().packed(q, k, v, cu, window=50)
    for a, b in ((0, 100), (100, n)):
        want, bound = reference(q[a:b], k[a:b], v[a:b], 0, None, 50, D ** -0.5, dtype)
        close(out[a:b], want, bound)
    kp = torch.randn(8, 16, 1, D, generator=g, device="cuda").to(_dt(dtype)).expand(8, 16, KH, D)
    table = torch.tensor([[3, 1, 7]], dtype=torch.int32, device="cuda")
    for new in (1, 40):
        cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        out = handle().paged(q[:new], kp, kp, table, cu, torch.tensor([45], dtype=torch.int32, device="cuda"))
        want, bound = reference(q[:new], gathered(kp, table, 0, 45), gathered(kp, table, 0, 45), 45 - new, None, 0, D ** -0.5, dtype)
        close(out, want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_unseen_keys_have_no_part(dtype, D):
    """NaN and infinities in K and V of positions that some rows do not see
    stay out of those rows, and reach the others."""
    torch = _torch()
    n, H, KH = 300, 4, 2
    g = gen(21)
    q, k, v = (torch.randn(n, h, D, generator=g, device="cuda").to(_dt(dtype)) for h in (H, KH, KH))
    v[37, 0, 3] = float("nan")
    v[200, 1, 5] = float("inf")
    v[299, 0, :] = float("-inf")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for window in (0, 40):
        out = handle().packed(q, k, v, cu, window=window)
        want, bound = reference(q, k, v, 0, None, window, D ** -0.5, dtype)
        close(out, want, bound)
    q[5, 1] = float("nan")
    k[250] = float("nan")
    clean = handle().packed(q, k, v, cu)
    assert torch.isnan(clean[5, 1].float()).all()
    assert torch.isfinite(clean[:5].float()).all() and torch.isfinite(clean[6:37].float()).all()
    assert torch.isfinite(clean[:200, 2].float()).all() and torch.isnan(clean[250:].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [2, 3, 6])
def test_unseen_keys_have_no_part_with_few_rows(dtype, D, new):
    """The same through the pages, a few new tokens a request: infinities and
    NaN in the last positions, which the first of the new rows do not see."""
    reqs = [(300, new), (40, new), (900, new)]
    q, kp, vp, table, cu, kv = make_paged(reqs, 16, 8, 4, D, dtype, 61)
    for b, (total, _) in enumerate(reqs):
        for back, head, x, val in ((1, 0, 3, "inf"), (new, 1, 5, "-inf"), (new - 1, 2, 7, "nan"), (1, 3, slice(None), "inf"),
                                   (20, 3, 2, "-inf")):
            p = total - back
            vp[int(table[b, p // 16]), p % 16, head, x] = float(val)
    for window in (0, 7):
        out = handle().paged(q, kp, vp, table, cu, kv, window=window)
        for b, (total, n) in enumerate(reqs):
            r = slice(int(cu[b]), int(cu[b + 1]))
            want, bound = reference(q[r], gathered(kp, table, b, total), gathered(vp, table, b, total), total - n, None,
                                    window, D ** -0.5, dtype)
            close(out[r], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores far apart: the running maximum moves, weights underflow."""
    torch = _torch()
    n, H, D = 400, 2, 64
    g = gen(5)
    q, k, v = (torch.randn(n, H, D, generator=g, device="cuda") for _ in range(3))
    k = k * torch.linspace(0.1, 6.0, n, device="cuda")[:, None, None]
    q, k, v = (x.to(_dt(dtype)) for x in (q * 4, k, v))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    sk = torch.tensor([300.0, -300.0], device="cuda")
    for s in (None, sk):
        out = handle().packed(q, k, v, cu, sinks=s)
        want, bound = reference(q, k, v, 0, s, 0, D ** -0.5, dtype)
        close(out, want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_keys_of_weight_zero_first(dtype, D):
    """Scores of -inf for the first 64 positions: as if they were not there."""
    torch = _torch()
    q, kp, vp, table, cu, kv = make_paged([(700, 300), (400, 3)], 16, 4, 2, D, dtype, 31)
    q[..., 0] = 1.0
    keys = [gathered(kp, table, b, n) for b, n in ((0, 700), (1, 400))]
    vals = [gathered(vp, table, b, n) for b, n in ((0, 700), (1, 400))]
    for b in range(2):
        kp[table[b, :4].long(), :, :, 0] = float("-inf")
    out = handle().paged(q, kp, vp, table, cu, kv)
    for b, (total, new) in enumerate([(700, 300), (400, 3)]):
        want, bound = reference(q[int(cu[b]):int(cu[b + 1])], keys[b][64:], vals[b][64:], total - new - 64, None, 0,
                                D ** -0.5, dtype)
        close(out[int(cu[b]):int(cu[b + 1])], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 150])
def test_scores_that_grow_late(dtype, window):
    """A request's last keys outweigh the earlier ones by more than the types'
    range, within tiles that all rows see and within those that some do not."""
    torch = _torch()
    n, H, D = 900, 4, 64
    g = gen(8)
    q, k, v = (torch.randn(n, h, D, generator=g, device="cuda") for h in (H, 2, 2))
    k = k * torch.where(torch.arange(n, device="cuda") % 97 > 80, 4.0, 0.05)[:, None, None]
    q, k, v = (x.to(_dt(dtype)) for x in (q * 4, k, v))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = handle().packed(q, k, v, cu, window=window)
    want, bound = reference(q, k, v, 0, None, window, D ** -0.5, dtype)
    close(out, want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3])
def test_scores_that_grow_within_the_first_tile(dtype, D, group):
    """Of the first 128 keys one group of 32 outweighs the groups before it by
    2^10, with the groups' weights written one after another: what is written
    has to follow the new reference.  All rows that see the tile whole, and
    those that see a part."""
    torch = _torch()
    n, H, KH = 420, 4, 2
    g = gen(40 + group)
    q, k, v = (torch.randn(n, h, D, generator=g, device="cuda") for h in (H, KH, KH))
    k = k * 0.25
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[32 * group:, :, 0] = 10 * math.log(2) * math.sqrt(D) / 8
    q, k, v = (x.to(_dt(dtype)) for x in (q, k, v))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for window in (0, 140):
        out = handle().packed(q, k, v, cu, window=window)
        want, bound = reference(q, k, v, 0, None, window, D ** -0.5, dtype)
        close(out, want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hidden", [32, 128, 200])
@pytest.mark.parametrize("off", [0, 30, -29, 150, -150])
def test_lowest_values_first(dtype, D, hidden, off):
    """A request's first keys have f16's lowest value as their score's factor (the
    usual mask): rows that see others give those the weights they have alone,
    wherever their scores lie (2^off), and the first rows, which see none
    other, the mean."""
    torch = _torch()
    reqs = [(700, 300), (400, 3), (520, 520)]
    q, kp, vp, table, cu, kv = make_paged(reqs, 16, 4, 2, D, dtype, 51)
    q[..., 0], q[..., 1] = 65504.0, 8.0
    for b, (total, _) in enumerate(reqs):
        pos = torch.arange(total, device="cuda")
        at = table[b, pos // 16].long(), pos % 16
        kk = kp[at]
        kk[..., 0] = 0.0
        kk[..., 1] = off * math.log(2) * math.sqrt(D) / 8
        kk[:hidden] = 0.0
        kk[:hidden, :, 0] = -65504.0
        kp[at] = kk
    for window in (0, 250):
        out = handle().paged(q, kp, vp, table, cu, kv, window=window)
        for b, (total, new) in enumerate(reqs):
            r = slice(int(cu[b]), int(cu[b + 1]))
            want, bound = reference(q[r], gathered(kp, table, b, total), gathered(vp, table, b, total), total - new, None,
                                    window, D ** -0.5, dtype)
            close(out[r], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 130])
def test_only_lowest_values(dtype, D, new):
    """Every key has the type's lowest value as its score's factor: the mean of
    V, with few rows and many.  The scores are alike, so only weights of 1, their
    sums and the result are rounded."""
    torch = _torch()
    reqs = [(new, new), (300, new)]
    q, kp, vp, table, cu, kv = make_paged(reqs, 16, 8, 4, D, dtype, 55, garbage=False)
    q[..., 0] = 65504.0 if dtype == "f16" else 1.0
    kp.zero_()
    kp[..., 0] = torch.finfo(_dt(dtype)).min
    out = handle().paged(q, kp, vp, table, cu, kv)
    for b, (total, n) in enumerate(reqs):
        r = slice(int(cu[b]), int(cu[b + 1]))
        k = torch.zeros(total, 4, D, device="cuda")
        want, bound = reference(q[r] * 0, k, gathered(vp, table, b, total), total - n, None, 0, D ** -0.5, dtype)
        close(out[r], want, bound)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_contexts_weigh_old_and_new_keys_alike(dtype):
    """One early key against 131,071 later ones of the same total weight, in
    hundreds of tiles a warp that all leave the maximum as it is: a factor
    beside 1 at each of them would add up (5e-6 a tile to 1e-3)."""
    torch = _torch()
    B, L, D, G, page = 296, 1 << 17, 8, 4, 64
    k = torch.zeros(L // page, page, 1, D, device="cuda")
    v = torch.full_like(k, -1.0)
    k[..., 0], k[..., 1] = 100.0, -10.0
    k[0, 0, :, 1], v[0, 0] = 0.0, 1.0
    table = torch.arange(L // page, dtype=torch.int32, device="cuda").expand(B, -1).contiguous()
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    kv = torch.full((B,), L, dtype=torch.int32, device="cuda")
    q, k, v = (x.to(_dt(dtype)) for x in (torch.ones(B, G, D, device="cuda"), k, v))
    for scale in (1.171, 1.1755, 1.18, 1.1843):
        out = handle().paged(q, k, v, table, cu, kv, scale=scale)
        handle().check()
        want, bound = reference(q[:1], k.flatten(0, 1), v.flatten(0, 1), L - 1, None, 0, scale, dtype)
        close(out, want.expand(out.shape), bound.expand(out.shape))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 3])
def test_few_rows_lose_nothing_in_the_weights(dtype, D, new):
    """With few rows the weights keep what their rounding leaves: of the bound
    the type's part falls on the result alone (u |out|), the rest (2^-14 A) on
    the weights' second rounding (2^-16 A bf16), sums and exponentials."""
    reqs = [(5000, new), (300, new), (17, new)]
    q, kp, vp, table, cu, kv = make_paged(reqs, 16, 16, 4, D, dtype, 71)
    out = handle().paged(q, kp, vp, table, cu, kv)
    for b, (total, n) in enumerate(reqs):
        r = slice(int(cu[b]), int(cu[b + 1]))
        k, v = gathered(kp, table, b, total), gathered(vp, table, b, total)
        want, _ = reference(q[r], k, v, total - n, None, 0, D ** -0.5, dtype)
        A, _ = reference(q[r], k, v.abs(), total - n, None, 0, D ** -0.5, dtype)
        tiny = 2.0 ** -25 if dtype == "f16" else 0.0
        close(out[r], want, (U[dtype] * want.abs() + 2.0 ** -14 * A + tiny) * 1.02 + 1e-30)


def test_same_inputs_same_bits():
    """Items split between blocks are joined in a fixed order."""
    torch = _torch()
    for dtype in DTYPES:
        for reqs in ([(5000, 1), (3000, 1), (70, 1)], [(5000, 200), (900, 33)]):
            q, kp, vp, table, cu, kv = make_paged(reqs, 16, 16, 2, 64, dtype, 4)
            first = handle().paged(q, kp, vp, table, cu, kv)
            for _ in range(5):
                assert torch.equal(handle().paged(q, kp, vp, table, cu, kv).view(torch.uint8), first.view(torch.uint8))


def test_side_stream_and_graph():
    """The calls follow the stream they are given, and can be captured."""
    torch = _torch()
    from picchio_b200 import Attention, kv_store, kv_tables
    reqs = [(700, 1), (33, 1), (260, 20)]
    q, kp, vp, table, cu, kv = make_paged(reqs, 16, 16, 2, 64, "bf16", 8, garbage=False)
    want = handle().paged(q, kp, vp, table, cu, kv)
    side = torch.cuda.Stream()
    att = Attention()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = att.paged(q, kp, vp, table, cu, kv)
    side.synchronize()
    assert torch.equal(got, want)
    got = att.paged(q, kp, vp, table, cu, kv, stream=side)
    side.synchronize()
    assert torch.equal(got, want)

    k = torch.randn(22, 2, 64, device="cuda").bfloat16()
    free, n_free = torch.arange(5, dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    held = torch.tensor([700, 33, 260], dtype=torch.int32, device="cuda") - torch.tensor([1, 1, 20], dtype=torch.int32, device="cuda")
    new = torch.tensor([1, 1, 20], dtype=torch.int32, device="cuda")

    def step():
        t = kv_tables(held, new, table, free, n_free, page_size=16, n_tokens=22)
        kv_store(kp, vp, k, k, t.slots)
        return att.paged(q, kp, vp, table, t.cu_new, t.kv_len)

    with torch.cuda.stream(side):
        eager = step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
        out.zero_()
        graph.replay()
        side.synchronize()
        assert torch.equal(out, eager)


def test_one_handle_on_two_streams():
    """Calls on one handle from stream to stream follow one another: they share
    its workspace."""
    torch = _torch()
    from picchio_b200 import Attention
    att = Attention()
    sets = [make_paged(r, 16, 16, 2, 64, d, s) for s, (r, d) in enumerate(
        (([(9000, 1), (3000, 1)], "bf16"), ([(5000, 300), (900, 33)], "f16"), ([(7000, 2)], "f32"), ([(4000, 4)] * 5, "bf16")))]
    want = [handle().paged(*t) for t in sets]
    streams = [torch.cuda.Stream() for _ in range(3)] + [torch.cuda.current_stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(24):
        s = streams[i % 4]
        if i % 3:
            got.append(att.paged(*sets[i % 4], stream=s if i % 2 else s.cuda_stream))
        else:
            with torch.cuda.stream(s):
                got.append(att.paged(*sets[i % 4]))
    torch.cuda.synchronize()
    att.check()
    for i, g in enumerate(got):
        assert torch.equal(g.view(torch.uint8), want[i % 4].view(torch.uint8)), i
    # a graph of a call, beside calls on other streams before and after it
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = att.paged(*sets[0])
    again = att.paged(*sets[1])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(again, want[1])


# ---- tables and store ---------------------------------------------------------


def plain_tables(kv, new, table, free, n_free, page, n_tokens):
    """Request by request, as the header states it."""
    table, free = [list(r) for r in table], list(free)
    kv = [max(x, 0) for x in kv]
    width, cap = len(table[0]), len(free)
    at = n_free
    for b, n in enumerate(new):
        if n < 0:
            for j in range(min(-(-kv[b] // page), width)):
                if at < cap:
                    free[at] = table[b][j]
                at += 1
    avail = min(at, cap)
    kv_end, cu, served, pos, slot = [], [0], [], [], []
    need = toks = used = 0
    for b, n in enumerate(new):
        fits = n >= 0 and kv[b] + n <= width * page
        held = -(-kv[b] // page)
        want = -(-(kv[b] + n) // page) - held if fits else 0
        need += want
        toks += n if fits else 0
        ok = fits and (want == 0 or need <= avail) and (n == 0 or toks <= n_tokens)
        if ok:
            for j in range(want):
                table[b][held + j] = free[avail - 1 - used - j]
            used += want
            for p in range(kv[b], kv[b] + n):
                pos.append(p)
                slot.append(table[b][p // page] * page + p % page)
        kv_end.append(0 if n < 0 else kv[b] + n if ok else kv[b])
        served.append(int(ok))
        cu.append(len(pos))
    fill = n_tokens - len(pos)
    return table, free, dict(kv_len=kv_end, cu_new=cu, served=served, n_free=[avail - used],
                             positions=pos + [-1] * fill, slots=slot + [-1] * fill)


def run_tables(kv, new, width, page, spare, n_tokens, cap_extra=0, seed=0):
    import random
    torch = _torch()
    from picchio_b200 import kv_tables
    r = random.Random(seed)
    have = [min(-(-max(x, 0) // page), width) for x in kv]
    ids = r.sample(range(sum(have) + spare + 5), sum(have) + spare)
    table, at = [], spare
    for h in have:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    free = ids[:spare] + [0] * (sum(have) + cap_extra)
    ti = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    t, f = ti(table), ti(free)
    want_t, want_f, want = plain_tables(kv, new, table, free, spare, page, n_tokens)
    for _ in range(2):  # the same inputs again: the same outputs
        got = kv_tables(ti(kv), ti(new), t, f, ti([spare]), page_size=page, n_tokens=n_tokens)
        for name, x in want.items():
            assert getattr(got, name).tolist() == x, name
        assert t.tolist() == want_t and f.tolist() == want_f
    assert got.slots.dtype == torch.int64


def test_tables_decode_and_pages():
    run_tables([0, 1, 15, 16, 17, 31, 32], [1] * 7, 4, 16, 6, 7)
    run_tables([0], [1], 1, 8, 1, 1)
    run_tables([0], [0], 1, 8, 0, 0)
    run_tables([5, 5], [0, -1], 2, 8, 0, 4)


def test_tables_without_requests():
    """A step with no request: no rows, the free pages as they were."""
    torch = _torch()
    from picchio_b200 import kv_tables
    ti = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for n in (0, 5, 3000):
        t = kv_tables(ti(), ti(), ti().view(0, 4), ti(7, 3, 9), ti(2), page_size=16, n_tokens=n)
        assert t.cu_new.tolist() == [0] and t.n_free.tolist() == [2] and t.kv_len.numel() == t.served.numel() == 0
        assert t.positions.tolist() == [-1] * n and t.slots.tolist() == [-1] * n


def test_tables_refusals_of_requests():
    run_tables([10, 60, 3, 64, 20], [7, 5, 0, 1, 100], 4, 16, 3, 200)      # past the table's width
    run_tables([16, 16, 16, 5, 16], [1, 40, 1, 1, 1], 8, 16, 3, 100)       # pages run out at the second
    run_tables([1, 1, 1, 1], [3, 4, 0, 5], 8, 16, 9, 8)                     # rows run out at the last
    run_tables([16, 50, 16, 30], [20, -1, 33, -1], 8, 16, 0, 100)           # served from ended requests' pages
    run_tables([-4, -1], [3, -1], 8, 16, 5, 4)                              # lengths below zero


def test_tables_sums_past_32_bits():
    """1024 requests that together ask for more rows than 32 bits count: none
    is served, whatever its sum would wrap to."""
    n = 1 << 21
    run_tables([0] * 1025, [n + 1] * 1024 + [3], 257, 8192, 1024 * 257 + 1, n)
    run_tables([0] * 1025, [2] + [n + 1] * 1023 + [3], 257, 8192, 1024 * 257 + 1, n)
    run_tables([2**31 - 1] * 3 + [1], [2**31 - 1, -1, 1, 1], 4, 16, 3, 4)


def test_tables_large_and_mixed():
    import random
    for seed in range(6):
        r = random.Random(seed)
        B = r.choice([33, 300, 1025, 2500])
        page = r.choice([8, 16, 24, 64])
        kv = [r.randint(0, 900) for _ in range(B)]
        new = [r.choice([1, 1, 1, 1, r.randint(0, 300), -1]) for _ in range(B)]
        width = r.randint(60, 900 // page + 60)
        total = sum(max(n, 0) for n in new)
        run_tables(kv, new, width, page, r.randint(0, 2 * B), r.choice([total, total // 2, total + 77]), seed=seed)


@pytest.mark.parametrize("src", DTYPES)
@pytest.mark.parametrize("dst", DTYPES)
@pytest.mark.parametrize("KH,D,page,n", [(8, 64, 16, 64), (1, 8, 8, 1), (2, 128, 32, 1000), (3, 40, 24, 77)])
def test_store(src, dst, KH, D, page, n):
    torch = _torch()
    from picchio_b200 import kv_store
    g = gen(n)
    pages = n // page + 3
    kp, vp = (torch.randn(pages, page, KH, D, generator=g, device="cuda").to(_dt(dst)) for _ in range(2))
    rows = torch.randn(n, 3 * KH * D + 8, generator=g, device="cuda").to(_dt(src))
    k, v = rows[:, KH * D:2 * KH * D].view(n, KH, D), rows[:, 2 * KH * D:3 * KH * D].view(n, KH, D)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    slots[::5] = -1
    if n > 8:
        slots[3] = pages * page  # outside the cache
        slots[6] = -(1 << 40)
    want = [kp.clone(), vp.clone()]
    keep = (slots >= 0) & (slots < pages * page)
    for w, r in zip(want, (k, v)):
        w.view(-1, KH, D)[slots[keep]] = r[keep].to(w.dtype)
    kv_store(kp, vp, k, v, slots)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    # a cache laid out heads first
    kt, vt = (torch.zeros(pages, KH, page, D, dtype=_dt(dst), device="cuda").permute(0, 2, 1, 3) for _ in range(2))
    kv_store(kt, vt, k, v, slots)
    at = slots[keep]
    assert torch.equal(kt[at // page, at % page], k[keep].to(kt.dtype))
    assert torch.equal(vt[at // page, at % page], v[keep].to(kt.dtype))


# ---- refusals ------------------------------------------------------------------


def test_attention_refusals():
    torch = _torch()
    from picchio_b200 import PicchioError, kv_store, kv_tables
    q, kp, vp, table, cu, kv = make_paged([(20, 2)], 16, 4, 2, 64, "bf16", 1)
    a = handle()
    with pytest.raises(ValueError):
        a.paged(q.double(), kp, vp, table, cu, kv)
    with pytest.raises(ValueError):
        a.paged(q, kp, vp[:-1], table, cu, kv)
    with pytest.raises(ValueError):
        a.paged(q, kp, vp, table.long(), cu, kv)
    with pytest.raises(ValueError):
        a.paged(q, kp, vp, table, cu, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        a.paged(q.cpu(), kp, vp, table, cu, kv)
    with pytest.raises(ValueError):
        a.paged(q, kp, vp, table, cu, kv, sinks=torch.zeros(3, device="cuda"))
    with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
        a.paged(q.half(), kp, vp, table, cu, kv)  # q and cache of two types
    with pytest.raises(PicchioError, match="PC_ERR_INVALID_ARG"):
        a.paged(q[:, :3], kp, vp, table, cu, kv)  # 3 heads over 2
    with pytest.raises(PicchioError, match="PC_ERR_INVALID_ARG"):
        a.paged(q, kp, vp, table, cu, kv, window=-1)
    with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
        a.paged(q[..., :60], kp[..., :60], vp[..., :60], table, cu, kv)  # head_dim not a multiple of 8
    with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
        a.paged(q, kp[:, :4], vp[:, :4], table, cu, kv)  # pages of 4
    big = torch.zeros(2, 4, 136, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
        a.packed(big, big, big, cu)
    off = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 4, 64)
    with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
        a.packed(off, off, off, cu)  # not on a 16-byte boundary
    with pytest.raises(ValueError):
        a.packed(q, q[:1], q[:1], cu)
    ti = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
        kv_tables(ti(1), ti(1), ti([1]).view(1, 1), ti(1, 2), ti(2), page_size=12, n_tokens=1)
    with pytest.raises(ValueError):
        kv_tables(ti(1), ti(1, 2), ti([1]).view(1, 1), ti(1, 2), ti(2), page_size=16, n_tokens=1)
    with pytest.raises(ValueError):
        kv_store(kp, vp, q, q, torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        kv_store(kp, vp, q[:, :2], q[:, :2], torch.zeros(2, dtype=torch.int32, device="cuda"))
    empty = q[:0]
    assert a.paged(empty, kp, vp, table, ti(0, 0), kv).shape == (0, 4, 64)


def test_numbers_out_of_every_range_are_refused():
    """Numbers that a C int or float does not hold, and a step of more rows
    than the tables count, by the library's own errors."""
    torch = _torch()
    from picchio_b200 import PicchioError, kv_tables
    q, kp, vp, table, cu, kv = make_paged([(20, 2)], 16, 4, 2, 64, "bf16", 1)
    ti = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for window in (-(1 << 40), -5):
        with pytest.raises(PicchioError, match="PC_ERR_INVALID_ARG"):
            handle().paged(q, kp, vp, table, cu, kv, window=window)
    for scale in (1e300, -1e300, float("inf"), float("nan"), 0.0):
        with pytest.raises(PicchioError, match="PC_ERR_INVALID_ARG"):
            handle().paged(q, kp, vp, table, cu, kv, scale=scale)
    for page in (1 << 40, -(1 << 40)):
        with pytest.raises(PicchioError, match="PC_ERR_FORMAT"):
            kv_tables(ti(1), ti(1), ti([1]).view(1, 1), ti(1, 2), ti(2), page_size=page, n_tokens=1)
    for n in (-1, (1 << 28) + 1, 1 << 40):
        with pytest.raises(ValueError):
            kv_tables(ti(1), ti(1), ti([1]).view(1, 1), ti(1, 2), ti(2), page_size=16, n_tokens=n)
