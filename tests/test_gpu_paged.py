"""The paged cache's operators (include/webgllm_paged.h) against plain 64-bit
forms (tests/paged_reference.py), within bounds derived from their arithmetic."""
import ctypes
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import paged_reference as R  # noqa: E402
import webgllm_b200 as wg  # noqa: E402
from webgllm_b200 import _lib, paged, q4  # noqa: E402
from webgllm_b200.speculative import spec_sample  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def p_eps(dtype, rows, batch, H, Hkv):
    """One 16-bit rounding of P: the coarsest any of the kernels makes."""
    return torch.finfo(dtype).eps / 2


def make(counts, pos, H, Hkv, Dh, page, dtype, seed=0, window=0, sinks=0, fill=float("nan"), freed=False):
    """Queries and pages: only what some row sees holds numbers, the rest `fill`."""
    g = gen(seed)

    def live(b):
        n, p = counts[b], pos[b]
        ws = max(0, p - window + 1) if window else 0
        if not freed or ws <= sinks:
            return [(0, max(0, p + n))] if n else []
        return [(0, sinks), (ws, p + n)] if n else []

    table, pages = R.layout(counts, pos, page, seed=seed, live=live)
    k = torch.full((pages, Hkv, page, Dh), fill, dtype=dtype, device="cuda")
    v = torch.full_like(k, fill)
    for b in range(len(counts)):
        for a, e in live(b):
            for j in range(a // page * page, e, page):
                pg, hi = table[b, j // page], min(page, e - j)
                lo = max(0, a - j)
                k[pg, :, lo:hi] = torch.randn((Hkv, hi - lo, Dh), generator=g, device="cuda").to(dtype)
                v[pg, :, lo:hi] = torch.randn((Hkv, hi - lo, Dh), generator=g, device="cuda").to(dtype)
    q = (torch.randn((sum(counts), H, Dh), generator=g, device="cuda") * (1.5 / Dh ** 0.5)).to(dtype)
    return q, k, v, table


def starts(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def run(q, k, v, table, counts, pos, window=0, sinks=0, ragged=None, **kw):
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    if ragged is None:
        ragged = len(set(counts)) > 1
    return paged.attention_paged(q, p, k, v, table, window=window, sinks=sinks,
                                 row_start=starts(counts) if ragged else None, **kw)


def check(out, q, k, v, table, counts, pos, window=0, sinks=0):
    wg.context().sync()  # no complaint from the device
    ref, bound = R.attention(q, k, v, table, counts, pos, window, sinks)
    keys = max([1] + [n + p for n, p in zip(counts, pos)])
    if window:
        keys = min(keys, window + sinks)
    tol = R.attention_tolerance(q.dtype, ref, bound, q.shape[2], keys, p_eps(q.dtype, 0, 0, 0, 0))
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.2f} of the bound"


CASES = [
    # counts, pos, H, Hkv, Dh, page, window, sinks, dtype
    ([1], [0], 4, 4, 64, 16, 0, 0, F16),                        # one key
    ([1], [255], 32, 4, 64, 16, 0, 0, F16),
    ([1], [256], 32, 8, 128, 64, 0, 0, BF16),
    ([1] * 5, [0, 63, 64, 65, 1000], 8, 2, 128, 64, 0, 0, F16),  # tile borders
    ([1] * 3, [15, 16, 700], 7, 1, 64, 48, 0, 0, BF16),          # MQA, 7 heads, odd page
    ([1] * 2, [300, 5], 40, 2, 64, 32, 0, 0, F16),               # 20 heads a KV head: two row tiles
    ([1] * 2, [129, 511], 6, 3, 256, 16, 0, 0, F16),
    ([1], [3000], 16, 1, 256, 128, 0, 0, BF16),
    ([1], [5000], 8, 1, 128, 16, 0, 0, F16),                     # one unit over many CTAs
    ([5] * 4, [0, 1, 500, 1234], 32, 8, 128, 64, 0, 0, F16),     # verify rows
    ([3] * 3, [61, 62, 63], 24, 8, 64, 32, 0, 0, BF16),
    ([2, 0, 7, 1, 0], [10, 99, 200, 0, 5], 8, 4, 64, 80, 0, 0, F16),  # ragged, empty sequences
    ([1] * 3, [0, 40, 2000], 8, 2, 64, 16, 1, 0, F16),           # a row that sees itself only
    ([1] * 4, [3, 63, 64, 3000], 8, 2, 128, 64, 64, 4, F16),
    ([1] * 4, [100, 130, 131, 900], 4, 4, 64, 16, 128, 70, BF16),  # sinks past a tile
    ([6] * 3, [0, 250, 777], 8, 2, 64, 48, 100, 3, F16),         # window edges differ by row
    ([4, 1, 9], [500, 2, 64], 12, 4, 128, 32, 33, 1, BF16),
    ([17], [0], 4, 2, 64, 16, 0, 0, F16),                        # many rows, little work: the split kernel
    ([64], [0], 32, 8, 128, 64, 0, 0, F16),
    ([130], [0], 8, 2, 128, 16, 0, 0, BF16),
    ([257], [100], 6, 3, 64, 48, 0, 0, F16),
    ([100, 1, 0, 300], [0, 50, 7, 129], 8, 2, 64, 32, 0, 0, BF16),
    ([200], [1000], 8, 8, 128, 128, 0, 0, F16),
    ([150], [300], 4, 2, 256, 64, 0, 0, F16),
    ([300], [0], 8, 2, 128, 64, 50, 0, F16),
    ([260], [700], 14, 2, 64, 16, 129, 5, BF16),
    ([333, 40], [1, 900], 8, 1, 128, 32, 200, 130, F16),
    ([140], [60], 2, 1, 256, 16, 64, 4, BF16),
    # prompts: work enough for the tensor-core kernel
    ([130], [0], 32, 8, 128, 64, 0, 0, F16),
    ([300], [0], 32, 8, 64, 16, 0, 0, BF16),
    ([200], [1000], 32, 32, 128, 128, 0, 0, F16),                # one head a KV head: 256 rows a unit
    ([65] * 4, [0, 1, 63, 500], 16, 4, 128, 48, 0, 0, BF16),
    ([100, 1, 0, 300], [0, 50, 7, 129], 56, 8, 64, 32, 0, 0, F16),  # 7 heads: 126 of a tile's 128 rows
    ([257], [100], 24, 8, 64, 80, 0, 0, F16),
    ([80], [300], 32, 8, 256, 64, 0, 0, F16),
    ([33, 64], [0, 99], 40, 2, 256, 16, 0, 0, BF16),             # 20 heads a KV head
    ([40], [600], 128, 1, 128, 16, 0, 0, F16),                   # 128 heads: a row a tile
    ([300], [0], 32, 8, 128, 64, 50, 0, F16),                    # windows: their edges, sinks, freed pages
    ([260], [700], 28, 4, 64, 16, 129, 5, BF16),
    ([333, 40], [1, 900], 24, 3, 128, 32, 200, 130, F16),
    ([140], [60], 32, 8, 256, 16, 64, 4, BF16),
    ([200] * 2, [5, 2000], 32, 8, 64, 64, 1, 1, F16),
    ([3] * 90, list(range(0, 1800, 20)), 32, 8, 128, 16, 0, 0, F16),  # many short ones
]


@pytest.mark.parametrize("counts,pos,H,Hkv,Dh,page,window,sinks,dtype", CASES)
def test_attention(counts, pos, H, Hkv, Dh, page, window, sinks, dtype):
    # everything that no row sees is NaN: other pages, the ends of pages
    q, k, v, table = make(counts, pos, H, Hkv, Dh, page, dtype, seed=H + Dh, window=window, sinks=sinks, freed=True)
    out = run(q, k, v, table, counts, pos, window, sinks)
    check(out, q, k, v, table, counts, pos, window, sinks)
    again = run(q, k, v, table, counts, pos, window, sinks, ragged=True)
    assert torch.equal(out, again)  # the same bits, also with explicit row starts


@pytest.mark.parametrize("rows,Dh,page", [(4, 64, 16), (5, 128, 64), (3, 256, 32), (100, 64, 32), (140, 128, 64),
                                          (70, 256, 16)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_what_later_rows_see_does_not_touch_earlier_ones(rows, Dh, page, dtype, bad):
    """A key / value of position p holds inf or NaN: rows before p are exact,
    and so are rows whose window has left it behind."""
    window, pos, hot = 24, 37, 37 + rows // 2
    # (64 heads: the longer ones go to the tensor-core kernel)
    q, k, v, table = make([rows], [pos], 64, 32, Dh, page, dtype, seed=rows, window=window, sinks=2)
    clean_k, clean_v = k.clone(), v.clone()
    pg = table[0, hot // page]
    k[pg, :, hot % page] = bad
    v[pg, :, hot % page, ::3] = bad
    out = run(q, k, v, table, [rows], [pos], window, 2)
    wg.context().sync()
    ref, bound = R.attention(q, clean_k, clean_v, table, [rows], [pos], window, 2)
    tol = R.attention_tolerance(dtype, ref, bound, Dh, window + 2, p_eps(dtype, 0, 0, 0, 0))
    i = torch.arange(pos, pos + rows, device="cuda")
    clear = (i < hot) | (i - window >= hot)
    assert clear.any() and (~clear).any()
    assert ((out.double() - ref).abs() <= tol)[clear].all()
    assert not torch.isfinite(out[~clear]).all()


def test_rows_that_see_nothing_and_rows_of_nobody():
    H, Hkv, Dh, page = 8, 2, 64, 16
    q, k, v, table = make([3, 3], [5, 40], H, Hkv, Dh, page, F16)
    # sequence 1 padded: positions -2, -1, 0
    pos = torch.tensor([5, -2], dtype=torch.int32, device="cuda")
    out = paged.attention_paged(q, pos, k, v, table)
    assert torch.equal(out[3:5], torch.zeros_like(out[3:5]))
    check(out[[0, 1, 2, 5]], q[[0, 1, 2, 5]], k, v, table, [3, 1], [5, 0])
    # rows 0 and 4.. belong to nobody
    out = torch.full_like(q, 7.0)
    rs = torch.tensor([1, 3, 4], dtype=torch.int32, device="cuda")
    paged.attention_paged(q, torch.tensor([6, -1], dtype=torch.int32, device="cuda"), k, v, table, row_start=rs, out=out)
    assert (out[[0, 4, 5]] == 7.0).all() and not out[3].any()
    check(out[1:3], q[1:3], k, v, table, [2, 0], [6, 0])


def test_a_long_prompt_with_padding_rows_first():
    H, Hkv, Dh, page = 32, 16, 128, 32
    q, k, v, table = make([200], [0], H, Hkv, Dh, page, F16)
    out = paged.attention_paged(q, torch.tensor([-130], dtype=torch.int32, device="cuda"), k, v, table)
    assert not out[:130].any()
    check(out[130:], q[130:], k, v, table, [70], [0])


@pytest.mark.parametrize("rows", [1, 3, 160])
def test_extreme_positions(rows):
    """The first and last positions an int32 holds: padding, and rows past the
    end of their table, which see all of it (or nothing through a window)."""
    H, Hkv, Dh, page, n = 32, 16, 128, 16, 64
    low, high = -2 ** 31, 2 ** 31 - 1
    # (every row of a sequence at `high` sees the whole table: 64 positions of data)
    q, k, v, table = make([1] * (3 * rows), [n - 1] * (3 * rows), H, Hkv, Dh, page, F16)
    table = table[[0, rows, 2 * rows]].contiguous()
    pos = torch.tensor([low, high, high - rows + 1], dtype=torch.int32, device="cuda")
    out = paged.attention_paged(q, pos, k, v, table)
    assert not out[:rows].any()
    check(out[rows:], q[rows:], k, v, table[[1] * rows + [2] * rows].contiguous(), [1] * (2 * rows), [n - 1] * (2 * rows))
    for window in (5, high):
        out = paged.attention_paged(q, pos, k, v, table, window=window)
        assert not out[:rows].any()
        if window == 5:
            assert not out.any()
    wg.context().sync()


def test_missing_pages_are_left_out_and_reported():
    counts, pos, H, Hkv, Dh, page = [1, 2], [100, 75], 8, 2, 64, 16
    for bad in (-1, 10 ** 6):
        q, k, v, table = make(counts, pos, H, Hkv, Dh, page, F16)
        table[0, 2] = bad
        table[1, 0] = bad
        out = run(q, k, v, table, counts, pos)
        with pytest.raises(wg.GpuError):
            wg.context().sync()
        check(out, q, k, v, table, counts, pos)
    # a long prompt
    q, k, v, table = make([300], [50], 64, 16, Dh, page, F16)
    table[0, 5] = -1
    out = run(q, k, v, table, [300], [50])
    with pytest.raises(wg.GpuError):
        wg.context().sync()
    check(out, q, k, v, table, [300], [50])


@pytest.mark.parametrize("order", ["rows_first", "layers", "k_next_to_v"])
def test_strided_pages(order):
    counts, pos, H, Hkv, Dh, page = [2, 2], [100, 75], 8, 2, 128, 32
    q, k, v, table = make(counts, pos, H, Hkv, Dh, page, F16)
    n = k.shape[0]
    if order == "rows_first":  # [pages][rows][heads][dims]
        k2 = k.transpose(1, 2).contiguous().transpose(1, 2)
        v2 = v.transpose(1, 2).contiguous().transpose(1, 2)
    elif order == "layers":  # layer 1 of [pages][layers][heads][rows][dims]
        both = torch.full((2, n, 3, Hkv, page, Dh), float("nan"), dtype=F16, device="cuda")
        both[0, :, 1], both[1, :, 1] = k, v
        k2, v2 = both[0, :, 1], both[1, :, 1]
    else:
        both = torch.stack([k, v], 3)  # [pages][heads][rows][2][dims]
        k2, v2 = both[..., 0, :], both[..., 1, :]
    out = run(q, k2, v2, table, counts, pos)
    assert torch.equal(out, run(q, k, v, table, counts, pos))
    # the append finds the same places
    qkv = torch.randn((4, (H + 2 * Hkv) * Dh), device="cuda")
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    a = paged.rope_kv_paged(qkv, p, k, v, table, heads=H)
    b = paged.rope_kv_paged(qkv, p, k2, v2, table, heads=H)
    assert torch.equal(a, b)
    assert torch.equal(k.nan_to_num(9.0), k2.nan_to_num(9.0)) and torch.equal(v.nan_to_num(9.0), v2.nan_to_num(9.0))


def high_keys(counts, pos, H, Hkv, Dh, page, dtype, highs, spread=0.5, seed=3):
    """Rows whose scores are `spread` N(0, 1) but for the keys of `highs`, which
    have score highs[j] and value 0."""
    g = gen(seed)
    table, pages = R.layout(counts, pos, page, seed=seed)
    n = counts[0] + pos[0]
    q = torch.full((counts[0], H, Dh), 0.25, dtype=dtype, device="cuda")
    k = torch.full((pages, Hkv, page, Dh), float("nan"), dtype=dtype, device="cuda")
    v = torch.full_like(k, float("nan"))
    j = torch.arange(n, device="cuda")
    kk = torch.randn((n, Hkv, Dh), generator=g, device="cuda") * (4 * spread / Dh ** 0.5)
    vv = torch.rand((n, Hkv, Dh), generator=g, device="cuda") + 0.5
    for at, score in highs.items():
        kk[at] = 4.0 * score / Dh
        vv[at] = 0.0
    at = table[0, j // page].long(), slice(None), j % page
    k[at], v[at] = kk.to(dtype), vv.to(dtype)
    return q, k, v, table


def check_high_keys(count, pos, H, Hkv, Dh, page, dtype, highs):
    """Within the bound of the other tests, which is relative to sum p |v|: here
    without the high keys' share. To that, for what fp16 rounds off below 2^-14:
    a share 2^-15 of sum p |v|, and 2^-26 of the largest value (1.5)."""
    q, k, v, table = high_keys([count], [pos], H, Hkv, Dh, page, dtype, highs)
    out = run(q, k, v, table, [count], [pos])
    wg.context().sync()
    ref, bound = R.attention(q, k, v, table, [count], [pos])
    tol = R.attention_tolerance(dtype, ref, bound, Dh, count + pos, p_eps(dtype, 0, 0, 0, 0))
    tol = tol + 2.0 ** -15 * bound[0] + 2.0 ** -26 * 1.5
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.2f} of the bound"


HIGHS = [
    {0: 14.0}, {0: 15.0}, {0: 16.0}, {0: 17.0}, {0: 20.0}, {0: 30.0}, {0: 80.0},  # a first token far above the rest
    {0: 17.0, 1500: 17.0}, {0: 17.0, 900: 40.0}, {700: 16.0},                     # one more later on
    {**{j: 12.0 for j in range(0, 2500, 64)}, 0: 20.0},                           # one in every tile
    {0: 80.0, **{j: 40.0 for j in range(64, 128)}},                               # two steps down
    {0: 17.0, 2000: 2.0 ** 12},                                                   # and far up
]


@pytest.mark.parametrize("count,pos,H,Hkv,Dh,dtype", [(200, 2800, 32, 8, 128, F16), (300, 2800, 32, 8, 64, F16),
                                                      (100, 2800, 32, 8, 256, F16), (200, 2800, 32, 8, 128, BF16)])
@pytest.mark.parametrize("highs", HIGHS, ids=lambda h: "-".join(f"{j}:{s:g}" for j, s in sorted(h.items())[:3]))
def test_prompt_keys_far_below_the_highest(count, pos, H, Hkv, Dh, dtype, highs):
    check_high_keys(count, pos, H, Hkv, Dh, 64, dtype, highs)


@pytest.mark.parametrize("count,pos,H,Hkv,Dh,dtype", [(1, 2999, 8, 2, 64, F16), (1, 2999, 8, 2, 128, F16),
                                                      (2, 2998, 4, 2, 256, F16), (5, 2995, 32, 8, 128, F16),
                                                      (1, 2999, 8, 2, 128, BF16)])
@pytest.mark.parametrize("highs", HIGHS, ids=lambda h: "-".join(f"{j}:{s:g}" for j, s in sorted(h.items())[:3]))
def test_decode_keys_far_below_the_highest(count, pos, H, Hkv, Dh, dtype, highs):
    check_high_keys(count, pos, H, Hkv, Dh, 16, dtype, highs)


@pytest.mark.parametrize("counts,H,Hkv,Dh", [([1] * 64, 8, 2, 64), ([1] * 64, 8, 4, 128), ([1] * 32, 4, 2, 256),
                                             ([5] * 8, 32, 8, 128), ([6] * 8, 32, 8, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_rows_hold_p_in_two_halves(counts, H, Hkv, Dh, dtype):
    """Values +1 and -1 that nearly cancel, and scores that are one exact product:
    what is left shows how P is rounded. With both halves (the second holds a
    remainder of at most 2^-11 or 2^-8 by half its last bit) it is off by 2^-23
    (fp16) or 2^-17 (bf16) of P, with one by 2^-11 or 2^-8: a kernel that drops a
    half, or the prompt kernel in these rows' place, is outside the bound, as the
    plain form with P in 16 bits is. The bound, relative to sum p |v| = 1: P; the
    exponent s log2 e - max + 14, below 16 in size and rounded once (2^-21, by ln 2),
    and exp2 (2^-21), both also in the row sum, and exp2 when warps are joined; fp32
    sums over the keys, twice."""
    B, n, pos, page = len(counts), counts[0], 15, 16
    g = gen(B + Dh)
    L = pos + n
    pages = B * 2
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(B, 2)
    q = torch.zeros((B * n, H, Dh), dtype=dtype, device="cuda")
    k = torch.zeros((pages, Hkv, page, Dh), dtype=dtype, device="cuda")
    q[..., 0] = 0.5
    k[..., 0] = torch.randint(-128, 129, k.shape[:3], generator=g, device="cuda") / 128.0  # (8 bits: exact in bf16)
    v = (torch.randint(0, 2, k.shape, generator=g, device="cuda") * 2 - 1).to(dtype)
    out = run(q, k, v, table, counts, [pos] * B)
    wg.context().sync()
    ref, (mass, _) = R.attention(q, k, v, table, counts, [pos] * B)
    half = torch.finfo(dtype).eps / 2
    c = (2.0 ** -23 if dtype is F16 else 2.0 ** -17) + 2 * 2.0 ** -21 + 3 * 2.0 ** -21 + 2 * L * 2.0 ** -24
    tol = half * (ref.abs() + c * mass) + c * mass
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.2f} of the bound"
    # the same with P in one number
    i = torch.arange(L, device="cuda")
    pg = table[:, i // page].long()
    kk = k[pg, :, i % page, 0].double().transpose(1, 2).repeat_interleave(H // Hkv, 1)  # [B][H][L]
    vv = v[pg, :, i % page].double().transpose(1, 2).repeat_interleave(H // Hkv, 1)
    s = (0.5 * kk)[:, None].masked_fill((i[None] > pos + torch.arange(n, device="cuda")[:, None])[None, :, None], -1e9)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    one = torch.einsum("bnhl,bhld->bnhd", p.to(dtype).double(), vv) / p.sum(-1, keepdim=True)
    assert ((one.reshape(ref.shape) - ref).abs() > 2 * tol).any()


@pytest.mark.parametrize("count,H,Hkv", [(1, 8, 2), (5, 32, 8), (200, 32, 8)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("score", [2.0 ** 15, 2.0 ** 22, -2.0 ** 23, 2.0 ** 23])
def test_scores_of_any_size(count, H, Hkv, dtype, score):
    """Half of the keys share one exact score far above the others': the result
    is their values' mean, however the reference of the exponentials is rounded.
    Off by P's rounding (the same for all), the sums' and the output's."""
    Dh, page, pos = 128, 16, 700
    q, k, v, table = make([count], [pos], H, Hkv, Dh, page, dtype, seed=count)
    q.fill_(16.0)
    top = torch.rand(k.shape[:3], generator=gen(5), device="cuda") < 0.5
    high, low = max(score, 0.0), min(score, 0.0)
    k.copy_(torch.where(top, high, low)[..., None] / (16 * Dh))
    out = run(q, k, v, table, [count], [pos])
    wg.context().sync()
    ref, (mass, _) = R.attention(q, k, v, table, [count], [pos])
    c = p_eps(dtype, 0, 0, 0, 0) + 2 * 2.0 ** -21 + 2 * (pos + count) * 2.0 ** -24
    assert ((out.double() - ref).abs() <= torch.finfo(dtype).eps / 2 * (ref.abs() + c * mass) + c * mass).all()


def test_offsets_past_32_bits():
    """Pages whose elements lie beyond 2^31 (and byte 2^32)."""
    Hkv, Dh, page = 8, 128, 64
    pages = (1 << 31) // (Hkv * Dh * page) + 40
    k = torch.empty((pages, Hkv, page, Dh), dtype=F16, device="cuda")
    v = torch.empty_like(k)
    k[-40:].normal_(generator=gen(1))
    v[-40:].normal_(generator=gen(2))
    for rows in (1, 150):
        n = 500
        table = torch.arange(pages - 10, pages, dtype=torch.int32, device="cuda").view(1, -1)
        q = (torch.randn((rows, 32, Dh), generator=gen(3), device="cuda") / 8).to(F16)
        out = run(q, k, v, table, [rows], [n - rows])
        check(out, q, k[-40:], v[-40:], table - (pages - 40), [rows], [n - rows])
    qkv = torch.randn((1, (16 + 2 * Hkv) * Dh), device="cuda")
    pos = torch.tensor([639], dtype=torch.int32, device="cuda")
    paged.rope_kv_paged(qkv, pos, k, v, table, heads=16)
    torch.cuda.synchronize()
    assert torch.equal(v[-1, :, 63], qkv.view(-1, Dh)[16 + Hkv:].half())


def test_shared_prefix_pages():
    counts, pos, H, Hkv, Dh, page = [1, 1, 1], [40, 47, 35], 4, 2, 64, 16
    q, k, v, table = make(counts, pos, H, Hkv, Dh, page, F16, fill=0.5)
    table[1, :2] = table[0, :2]
    table[2, :2] = table[0, :2]
    check(run(q, k, v, table, counts, pos), q, k, v, table, counts, pos)


def test_many_sequences():
    """More sequences than a CTA has threads, a few of them long."""
    B = 700
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 90, (B,), generator=g).tolist()
    pos[5], pos[400] = 3000, 1500
    counts = [1] * B
    q, k, v, table = make(counts, pos, 4, 2, 64, 16, F16, seed=3)
    check(run(q, k, v, table, counts, pos), q, k, v, table, counts, pos)


@pytest.mark.parametrize("rows", [1, 150])
def test_streams_and_graphs(rows):
    """On a side stream, captured, and two graphs replayed at once: each call
    has its own workspace."""
    counts, H, Hkv, Dh, page = [rows] * 2, 16, 2, 128, 64
    a = make(counts, [1500, 700], H, Hkv, Dh, page, F16, seed=1)
    b = make(counts, [900, 2222], H, Hkv, Dh, page, F16, seed=2)
    pa = torch.tensor([1500, 700], dtype=torch.int32, device="cuda")
    pb = torch.tensor([900, 2222], dtype=torch.int32, device="cuda")
    want = [paged.attention_paged(x[0], p, *x[1:]) for x, p in ((a, pa), (b, pb))]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for s, x, p in zip(side, (a, b), (pa, pb)):
        o = torch.empty_like(x[0])
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            paged.attention_paged(x[0], p, *x[1:], out=o)
        graphs.append(gr)
        outs.append(o)
    for _ in range(20):
        for s, gr, o in zip(side, graphs, outs):
            with torch.cuda.stream(s):
                o.zero_()
                gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    # the positions live on the device: a replay follows them
    pa -= 1
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], paged.attention_paged(a[0], pa, *a[1:]))


@pytest.mark.parametrize("counts,pos,H,Hkv,Dh,page,theta,norm,dtype", [
    ([1], [0], 4, 4, 64, 16, 1e4, False, F16),
    ([1] * 8, [0, 1, 63, 64, 640, 9999, 131071, 77], 32, 8, 128, 64, 5e5, False, F16),
    ([5, 0, 3, 17], [7, 1, 30000, 0], 24, 8, 64, 48, 1e6, True, BF16),
    ([33], [65520], 7, 1, 256, 32, 1e4, True, F16),
    ([300, 1], [0, 5], 14, 2, 64, 16, 5e5, True, F16),
    ([2, 2], [1048000, 3], 3, 3, 128, 128, 1e4, False, BF16),
])
def test_append(counts, pos, H, Hkv, Dh, page, theta, norm, dtype):
    g = gen(H + Dh)
    table, pages = R.layout(counts, pos, page, seed=H, live=lambda b: [(pos[b], pos[b] + counts[b])])
    rows = sum(counts)
    k = torch.full((pages, Hkv, page, Dh), 3.0, dtype=dtype, device="cuda")
    v = torch.full_like(k, 4.0)
    qkv = torch.randn((rows + 2, (H + 2 * Hkv) * Dh), generator=g, device="cuda")  # two rows of nobody
    qn = torch.rand(Dh, generator=g, device="cuda") + 0.5 if norm else None
    kn = torch.rand(Dh, generator=g, device="cuda") + 0.5 if norm else None
    out = torch.full((rows + 2, H, Dh), 5.0, dtype=dtype, device="cuda")
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    paged.rope_kv_paged(qkv, p, k, v, table, heads=H, theta=theta, q_norm=qn, k_norm=kn, row_start=starts(counts),
                        out=out)
    wg.context().sync()
    at = [(b, p + i) for b, (n, p) in enumerate(zip(counts, pos)) for i in range(n)]
    wq, wk, wv = R.rope(qkv[:rows], H, Hkv, Dh, [i for _, i in at], theta, qn, kn, 1e-5)
    assert ((out[:rows].double() - wq).abs() <= R.rope_tolerance(dtype, wq)).all()
    assert (out[rows:] == 5.0).all()
    b, i = torch.tensor(at, device="cuda").t()
    pg = table[b, i // page].long()
    assert ((k[pg, :, i % page].double() - wk).abs() <= R.rope_tolerance(dtype, wk)).all()
    assert torch.equal(v[pg, :, i % page], wv.to(dtype))
    k[pg, :, i % page] = 3.0
    v[pg, :, i % page] = 4.0
    assert (k == 3.0).all() and (v == 4.0).all()  # nothing else was written


def test_append_padding_and_missing_pages():
    H, Hkv, Dh, page = 4, 2, 64, 16
    table = torch.tensor([[0, -1, 2], [1, 9, 3]], dtype=torch.int32, device="cuda")
    k = torch.zeros((4, Hkv, page, Dh), dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.randn((6, (H + 2 * Hkv) * Dh), device="cuda")

    def call(pos, out=None):
        return paged.rope_kv_paged(qkv, torch.tensor(pos, dtype=torch.int32, device="cuda"), k, v, table, heads=H,
                                   out=out)

    q = call([-2, -3])  # positions -2, -1, 0 and -3, -2, -1: padding is no error
    wg.context().sync()
    assert not q[:2].any() and not q[3:].any() and q[2].any()
    assert v[0, :, 0].any() and not v[0, :, 1:].any() and not v[1:].any()
    v.zero_()
    # 14, 15 fit; 16 has no page; 46, 47 fit; 48 is past the table
    q = call([14, 46])
    with pytest.raises(wg.GpuError):
        wg.context().sync()
    wg.context().sync()
    assert q.any(-1).all()
    assert v[0, :, 14:].any(-1).all() and v[3, :, 14:].any(-1).all()
    assert not v[1].any() and not v[2].any()
    v.zero_()
    call([0, 16])  # sequence 1's page 9 does not exist
    with pytest.raises(wg.GpuError):
        wg.context().sync()
    assert not v[1:].any()


def test_append_in_a_graph_follows_positions():
    H, Hkv, Dh, page = 8, 2, 128, 64
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    k = torch.zeros((4, Hkv, page, Dh), dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.randn((2, (H + 2 * Hkv) * Dh), device="cuda")
    pos = torch.tensor([62, 0], dtype=torch.int32, device="cuda")
    out = torch.empty((2, H, Dh), dtype=BF16, device="cuda")
    paged.rope_kv_paged(qkv, pos, k, v, table, heads=H, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.rope_kv_paged(qkv, pos, k, v, table, heads=H, out=out)
        pos += 1
    k.zero_()
    v.zero_()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert v[0, :, 62:].any(-1).all() and v[1, :, 0].any(-1).all() and v[2, :, :3].any(-1).all()
    assert not v[1, :, 1:].any() and not v[2, :, 3:].any() and not v[3].any()


def test_c_level_refusals():
    """Argument checks of the C entry points (nothing is launched)."""
    L, c = _lib.lib(), wg.context()
    c.use_torch_stream()
    t = torch.zeros(4096, device="cuda")
    d = t.data_ptr()
    n = ctypes.c_size_t()
    assert L.wg_paged_attention_workspace(c.handle, 96, ctypes.byref(n)) == _lib.WG_INVALID_SHAPE
    assert L.wg_paged_attention_workspace(c.handle, 64, ctypes.byref(n)) == 0 and n.value > 0
    assert L.wg_paged_attention_workspace(c.handle, 64, None) == _lib.WG_INVALID_ARGUMENT

    def attend(rows=2, batch=2, H=4, Hkv=2, Dh=64, q=d, pos=d, out=d, ws=d, ws_bytes=n.value, window=0, sinks=0,
               k=d, v=d, table=d, dtype=_lib.WG_F16, pages=2, size=16, most=2, sp=0, sh=0, sr=0, kv=True, rs=None):
        s = _lib.wg_paged_kv(k, v, table, dtype, pages, size, most, sp, sh, sr)
        return L.wg_paged_attention(c.handle, q, rows, batch, rs, H, Hkv, Dh, pos, ctypes.byref(s) if kv else None,
                                    window, sinks, out, ws, ws_bytes)

    def append(rows=2, batch=2, H=4, Hkv=2, Dh=64, qkv=d, pos=d, out=d, theta=1e4, k=d, dtype=_lib.WG_F16, size=16,
               norm=None):
        s = _lib.wg_paged_kv(k, d, d, dtype, 2, size, 2, 0, 0, 0)
        return L.wg_paged_rope_kv(c.handle, qkv, rows, batch, None, H, Hkv, Dh, pos, theta, norm, None, 1e-5, out,
                                  ctypes.byref(s))

    A, S, U = _lib.WG_INVALID_ARGUMENT, _lib.WG_INVALID_SHAPE, _lib.WG_UNSUPPORTED
    for fn in (attend, append):
        for st, kw in [(S, dict(rows=3)), (S, dict(rows=-2)), (S, dict(batch=0)), (S, dict(H=3)), (S, dict(Hkv=0)),
                       (S, dict(Dh=96)), (S, dict(size=24)), (S, dict(size=0)), (A, dict(dtype=_lib.WG_F32)),
                       (A, dict(k=None)), (A, dict(k=d + 8)), (A, dict(pos=None)), (A, dict(out=None)),
                       (A, dict(out=d + 2)), (A, dict(pos=d + 2))]:
            assert fn(**kw) == st, (fn.__name__, kw)
        assert fn(rows=0) == 0
    for st, kw in [(A, dict(q=None)), (A, dict(q=d + 2)), (A, dict(ws=None)), (A, dict(ws=d + 4)),
                   (A, dict(ws_bytes=n.value - 1)), (A, dict(window=-1)), (A, dict(sinks=-1)), (A, dict(v=None)),
                   (A, dict(table=None)), (A, dict(kv=False)), (S, dict(pages=0)), (S, dict(most=0)),
                   (S, dict(most=1 << 28)), (S, dict(sp=4)), (S, dict(sh=-8)), (S, dict(sr=32)), (A, dict(rs=d + 1)),
                   (U, dict(rows=1 << 22, batch=1 << 20, most=1 << 20))]:
        assert attend(**kw) == st, kw
    assert attend(out=d + 2 * 2 * 4 * 64 - 16) == A and "overlap" in L.wg_last_error(c.handle).decode()
    assert attend(q=d + 16) == A and "overlap" in L.wg_last_error(c.handle).decode()
    for st, kw in [(A, dict(qkv=None)), (A, dict(qkv=d + 4)), (A, dict(theta=0.0)), (A, dict(theta=float("nan"))),
                   (A, dict(norm=d + 2)), (U, dict(rows=1 << 30, batch=1 << 20))]:
        assert append(**kw) == st, kw
    assert "wg_paged_rope_kv" in L.wg_last_error(c.handle).decode()


def test_overlapping_tensors_are_refused():
    """What a call writes shares no memory with what it reads in another order
    (nothing is launched)."""
    L, c = _lib.lib(), wg.context()
    c.use_torch_stream()
    t = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    d = t.data_ptr()
    n = ctypes.c_size_t()
    assert L.wg_paged_attention_workspace(c.handle, 64, ctypes.byref(n)) == 0
    pages = torch.zeros((2, 2, 2, 16, 64), dtype=F16, device="cuda")
    table = torch.tensor([[0, -1], [1, -1]], dtype=torch.int32, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    kv = _lib.wg_paged_kv(pages[0].data_ptr(), pages[1].data_ptr(), table.data_ptr(), _lib.WG_F16, 2, 16, 2, 0, 0, 0)
    A, qkv, q = _lib.WG_INVALID_ARGUMENT, 2 * 8 * 64 * 4, 2 * 4 * 64 * 2  # bytes of 2 rows of 4 + 2 x 2 heads

    def append(out):
        return L.wg_paged_rope_kv(c.handle, d + q, 2, 2, None, 4, 2, 64, pos.data_ptr(), 1e4, None, None, 1e-5, d + out,
                                  ctypes.byref(kv))

    def attend(ws):
        return L.wg_paged_attention(c.handle, d + 4096, 2, 2, None, 4, 2, 64, pos.data_ptr(), ctypes.byref(kv), 0, 0,
                                    d + 4096 + q, d + ws, n.value)

    for out in (16, q, q + qkv - 16):
        assert append(out) == A and "overlap" in L.wg_last_error(c.handle).decode()
    for ws in (16, 4096, 4096 + q, 4096 + 2 * q - 16):
        assert attend(ws) == A and "overlap" in L.wg_last_error(c.handle).decode()
    assert append(0) == 0 and append(q + qkv) == 0 and attend(4096 + 2 * q) == 0
    c.sync()


def test_another_current_stream_is_honoured():
    """Inputs made on a side stream are used in its order."""
    H, Hkv, Dh, page = 8, 2, 64, 16
    q, k, v, table = make([1], [500], H, Hkv, Dh, page, F16)
    want = run(q, k, v, table, [1], [500])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    q2 = torch.zeros_like(q)
    big = torch.zeros(1 << 28, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(5):
            big += 1.0  # keep the stream busy before q2 is written
        q2.copy_(q)
        out = run(q2, k, v, table, [1], [500])
    s.synchronize()
    assert torch.equal(out, want)


def test_native_and_python_calls_agree(monkeypatch):
    """The calls as one native step and through Python's code: the same bits;
    what the native step does not take, it leaves alone."""
    host = q4.host_calls()
    if host is None:
        pytest.skip("webgllm_b200._host is not built")
    g = gen(4)
    H, Hkv, Dh, page = 8, 2, 64, 16
    q, k, v, table = make([2, 3], [50, 70], H, Hkv, Dh, page, BF16)
    pos = torch.tensor([50, 70], dtype=torch.int32, device="cuda")
    rs = starts([2, 3])
    qkv = torch.randn((5, (H + 2 * Hkv) * Dh), generator=g, device="cuda")
    norm = torch.rand(Dh, generator=g, device="cuda")
    target = torch.randn((3, 4, 999), generator=g, device="cuda")
    draft = torch.randn((2, 4, 999), generator=g, device="cuda")
    drafts = torch.randint(0, 999, (4, 2), generator=g, device="cuda").to(torch.int32)
    u = torch.rand((4, 3), generator=g, device="cuda")
    ws = torch.empty(paged.workspace_bytes(0, Dh), dtype=torch.uint8, device="cuda")

    def everything():
        a = paged.rope_kv_paged(qkv, pos, k, v, table, heads=H, theta=1e6, q_norm=norm, eps=1e-6, row_start=rs)
        b = paged.attention_paged(a, pos, k, v, table, window=40, sinks=2, row_start=rs)
        c = paged.attention_paged(a, pos, k, v, table, row_start=rs, out=torch.empty_like(a), workspace=ws)
        return [a, b, c, k.clone(), v.clone(), spec_sample(target, draft, drafts, u, temperature=0.5),
                spec_sample(target[0], None, None, u[:, :1].contiguous())]

    native = everything()
    for name in ("webgllm_b200.paged", "webgllm_b200.speculative"):
        monkeypatch.setattr(f"{name}.host_calls", lambda: None)
    for x, y in zip(native, everything()):
        assert x.dtype == y.dtype and torch.equal(x.view(torch.int16 if x.dtype == BF16 else x.dtype),
                                                  y.view(torch.int16 if y.dtype == BF16 else y.dtype))
    out = torch.empty_like(q)
    assert host.attention_paged(q, pos, k, v, table, 0, 0, rs, out, None) is out
    for bad in [(q[..., :32], pos, k, v, table, 0, 0, rs, None, None), (q, pos.long(), k, v, table, 0, 0, rs, None, None),
                (q, pos, k, v[:, :, :8], table, 0, 0, rs, None, None), (q, pos, k, v, table, -1, 0, rs, None, None),
                (q, pos, k, v, table, 1 << 40, 0, rs, None, None), (q, pos, k, v, table, 0, 0, pos, None, None),
                (q, pos, k, v, table, 0, 0, rs, q, None), (q.cpu(), pos, k, v, table, 0, 0, rs, None, None),
                (q, pos, k, v, table, 0, 0, rs, None, ws[:64]), (q, pos, k.float(), v, table, 0, 0, rs, None, None),
                (q, pos, k, v, None, 0, 0, rs, None, None), (q, pos, k, v, table, 0, 0, rs, None), ()]:
        assert host.attention_paged(*bad) is None
    ctx = wg.context()
    with ctx.lock:  # another thread's call: left to the Python code, which waits
        assert host.attention_paged(q, pos, k, v, table, 0, 0, rs, None, None) is None
    assert host.attention_paged(q, pos, k, v, table, 0, 0, rs, None, None) is not None and not ctx.lock.locked()
    ctx.sync()


def test_calls_from_several_threads():
    """Threads on streams of their own: each call's work is on its thread's."""
    H, Hkv, Dh, page = 8, 2, 64, 16
    q, k, v, table = make([1] * 8, [300] * 8, H, Hkv, Dh, page, F16)
    pos = torch.full((8,), 300, dtype=torch.int32, device="cuda")
    want = paged.attention_paged(q, pos, k, v, table)
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(200):
                mine = q.clone()  # on this stream
                out = paged.attention_paged(mine, pos, k, v, table)
                mine.fill_(float("nan"))
            s.synchronize()
            if not torch.equal(out, want):
                wrong.append(out)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    wg.context().sync()
