"""wg_spec_sample against the definition in 64 bits (tests/paged_reference.py):
whole numbers, so equal."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import ctypes  # noqa: E402

import paged_reference as R  # noqa: E402
import webgllm_b200 as wg  # noqa: E402
from webgllm_b200 import _lib  # noqa: E402
from webgllm_b200.speculative import spec_sample  # noqa: E402


def make(B, k, V, noise, seed=0, spread=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = torch.randn((k + 1, B, V), generator=g, device="cuda") * spread
    u = torch.rand((B, k + 1), generator=g, device="cuda")
    if not k:
        return t, None, None, u
    d = t[:k] + noise * torch.randn((k, B, V), generator=g, device="cuda")
    drafts = torch.multinomial(torch.softmax(d.view(k * B, V), 1), 1, generator=g).view(k, B).t()
    return t, d, drafts.to(torch.int32).contiguous(), u


@pytest.mark.parametrize("B,k,V,noise,T", [
    (1, 0, 1, 0.0, 1.0), (3, 0, 2, 0.0, 0.5), (4, 0, 31, 0.0, 1.0), (5, 0, 4097, 0.0, 1.3), (8, 0, 32000, 0.0, 0.8),
    (2, 0, 128256, 0.0, 1.0), (4, 1, 1, 0.5, 1.0), (16, 2, 3, 1.0, 1.0), (9, 4, 1000, 0.5, 0.7),
    (7, 8, 2049, 0.2, 1.0), (3, 32, 515, 0.1, 1.0), (33, 5, 65543, 0.3, 0.9), (4, 4, 128256, 0.5, 1.0),
    (2, 3, 300001, 0.1, 1.0), (1, 1, 1 << 21, 1.0, 1.0), (6, 3, 5003, 1e-4, 1.0), (6, 3, 5003, 1e-7, 1.0),
    (4, 4, 777, 0.5, 0.01), (4, 4, 777, 0.5, 50.0),
])
def test_matches_the_definition(B, k, V, noise, T):
    t, d, drafts, u = make(B, k, V, noise, seed=B + V)
    got = spec_sample(t, d, drafts, u, temperature=T)
    wg.context().sync()
    assert torch.equal(got.cpu(), R.spec_picks(t, d, drafts, u, T))
    assert torch.equal(got, spec_sample(t, d, drafts, u, temperature=T))


def test_filtered_logits():
    """Tokens filtered by -inf (top-k) are never picked; a draft outside the
    target's filter is rejected."""
    t, d, drafts, u = make(32, 3, 4000, 0.5, seed=5)
    for x in (t, d):
        kth = x.topk(40, dim=2).values[..., -1:]
        x[x < kth] = -float("inf")
    drafts = torch.softmax(d, 2).argmax(2).t().to(torch.int32).contiguous()
    got = spec_sample(t, d, drafts, u)
    wg.context().sync()
    want = R.spec_picks(t, d, drafts, u, 1.0)
    assert torch.equal(got.cpu(), want)
    b, n = torch.arange(32), (want >= 0).sum(0) - 1
    assert torch.isfinite(t[n, b, got[n.cuda(), b.cuda()].long()]).all()


@pytest.mark.parametrize("top", [3e5, 2e8, 1e12, 1e30, 3e38, -1e30])
@pytest.mark.parametrize("T", [1.0, 1e-4])
def test_logits_of_any_size(top, T):
    """Finite logits however large: rows of three values, of which only the
    largest has probability, and drafts that have it in the draft."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    B, k, V = 24, 2, 3001
    values = sorted([top, top * (1 - 2.0 ** -10), -top])
    values = torch.tensor(values, device="cuda")
    t = values[torch.multinomial(torch.tensor([0.6, 0.1, 0.3], device="cuda").expand((k + 1) * B, 3), V,
                                 replacement=True, generator=g)].view(k + 1, B, V)
    d = values[torch.multinomial(torch.tensor([0.2, 0.1, 0.7], device="cuda").expand(k * B, 3), V,
                                 replacement=True, generator=g)].view(k, B, V)
    drafts = torch.multinomial((d == values[2]).float().view(k * B, V), 1, generator=g).view(k, B).t()
    drafts = drafts.to(torch.int32).contiguous()
    t[:, ::2].scatter_(2, drafts.t()[:, ::2, None].long().expand(k, B // 2, 1).contiguous(), top if top > 0 else -top)
    u = torch.rand((B, k + 1), generator=g, device="cuda")
    got = spec_sample(t, d, drafts, u, temperature=T)
    wg.context().sync()
    assert torch.equal(got.cpu(), R.spec_picks(t, d, drafts, u, T))


def test_the_ends_of_u():
    """u = 0 accepts whatever has probability and draws the first token that
    has; the largest u below one draws a token that has."""
    t, d, drafts, u = make(8, 2, 3001, 0.5, seed=9)
    t[:, :, :5] = -float("inf")
    t[:, :, -7:] = -float("inf")
    for value in (0.0, 1.0 - 2.0 ** -24):
        u.fill_(value)
        got = spec_sample(t, d, drafts, u)
        assert torch.equal(got.cpu(), R.spec_picks(t, d, drafts, u, 1.0))
    got = spec_sample(t[:1], None, None, torch.zeros((8, 1), device="cuda"))
    assert (got == 5).all()
    got = spec_sample(t[:1], None, None, torch.full((8, 1), 1.0, device="cuda"))  # taken as the largest below one
    assert (got >= 5).all() and (got < 3001 - 7).all()


def test_equal_distributions_are_always_accepted():
    t, _, _, u = make(16, 4, 2000, 0.0, seed=2)
    d = t[:4].clone()
    drafts = torch.randint(0, 2000, (16, 4), device="cuda", dtype=torch.int32)
    got = spec_sample(t, d, drafts, u)
    assert torch.equal(got[:4].t(), drafts)


def test_rejected_token_is_never_drawn():
    """Also where p - q leaves nothing but rounding: the picks applied by
    wg_spec_accept must stop at the drawn token."""
    V, B, k = 50, 64, 2
    t, _, _, u = make(B, k, V, 0.0, seed=4)
    d = t[:k].clone()
    drafts = torch.randint(0, V, (B, k), device="cuda", dtype=torch.int32)
    # the draft holds its token for a hair more likely than the target does
    for j in range(k):
        d[j].scatter_add_(1, drafts[:, j:j + 1].long(), torch.full((B, 1), 2e-6, device="cuda"))
    u[:, :k] = 1.0 - 2.0 ** -24
    got = spec_sample(t, d, drafts, u)
    wg.context().sync()
    assert torch.equal(got.cpu(), R.spec_picks(t, d, drafts, u, 1.0))
    n = (got >= 0).sum(0) - 1
    rejected = n < k
    assert rejected.any()
    b = torch.arange(B, device="cuda")
    assert (got[n, b][rejected] != drafts[b, n.clamp_max(k - 1)][rejected]).all()


def test_drafts_outside_the_vocabulary_are_rejected():
    t, d, drafts, u = make(4, 2, 100, 0.5, seed=3)
    drafts[0, 0], drafts[1, 0], drafts[2, 1] = -1, 100, 2 ** 31 - 1
    got = spec_sample(t, d, drafts, u)
    wg.context().sync()
    assert torch.equal(got.cpu(), R.spec_picks(t, d, drafts, u, 1.0))


@pytest.mark.parametrize("bad", ["nan", "inf", "none"])
@pytest.mark.parametrize("V", [1, 9, 40000])
def test_rows_without_probabilities_are_reported(bad, V):
    t, d, drafts, u = make(3, 1, V, 0.5, seed=1)
    drafts.zero_()
    if bad == "nan":
        t[:, 1, V // 2] = float("nan")
    elif bad == "inf":
        t[:, 1, V // 2] = float("inf")
    else:
        t[:, 1] = -float("inf")
    got = spec_sample(t, d, drafts, u)
    with pytest.raises(wg.GpuError):
        wg.context().sync()
    assert ((got[0] >= 0) & (got[0] < V)).all()
    ok = [0, 2]
    assert torch.equal(got.cpu()[:, ok], R.spec_picks(t[:, ok], d[:, ok], drafts[ok], u[ok], 1.0))


@pytest.mark.parametrize("bad", ["nan", "inf", "none"])
@pytest.mark.parametrize("V", [1, 9, 3000, 40000, 128256])
def test_plain_sampling_of_rows_without_probabilities(bad, V):
    t, _, _, u = make(5, 0, V, 0.0, seed=2)
    if bad == "nan":
        t[0, 3, V // 3] = float("nan")
    elif bad == "inf":
        t[0, 3, V - 1] = float("inf")
    else:
        t[0, 3] = -float("inf")
    t[0, 1, V // 2:] = -float("inf") if V > 1 else 0.0
    got = spec_sample(t, None, None, u)
    with pytest.raises(wg.GpuError):
        wg.context().sync()
    assert ((got >= 0) & (got < V)).all()
    ok = [0, 1, 2, 4]
    assert torch.equal(got.cpu()[:, ok], R.spec_picks(t[:, ok], None, None, u[ok], 1.0))


@pytest.mark.parametrize("V,k", [(32000, 0), (128256, 0), (128256, 1)])
def test_slices_without_weight_and_a_draw_on_their_border(V, k):
    """Runs of the vocabulary with the contents A B C none C B A none: u = 0.5
    draws on the border between the two C, whose running sum comes out an ulp
    higher or lower next to the run without weight, by the order of its additions.
    Each row gets one pick all the same: a neighbour of the border, or where the
    sum rounds past it, and the same one every time."""
    runs = {32000: 8, 128256: 16}[V]  # as many as CTAs share a row
    n = -(-V // runs)
    B = 18 if V > 32000 else 64
    g = torch.Generator(device="cuda")
    g.manual_seed(V + k)
    none = torch.full((B, n), -float("inf"), device="cuda")
    a, b, c = (none.clone().index_copy_(1, torch.tensor([i], device="cuda"), torch.randn((B, 1), generator=g, device="cuda"))
               for i in (3, n // 2, n - 200))
    row = torch.cat([a, b, c, none, c, b, a, none] + [none] * (runs - 8), 1)[:, :V]
    want = {2 * n + n - 200, 4 * n + n - 200}  # the two C
    t = row.expand(k + 1, B, V).contiguous()
    u = torch.full((B, k + 1), 0.5, device="cuda")
    d = drafts = None
    if k:  # a draft that the target keeps: the token is drawn from the last row
        d = torch.zeros((k, B, V), device="cuda")
        drafts = torch.full((B, k), 3, dtype=torch.int32, device="cuda")
    out = torch.full((k + 1, B), -7, dtype=torch.int32, device="cuda")
    spec_sample(t, d, drafts, u, out=out)
    wg.context().sync()
    assert set(out[k].tolist()) <= want
    for _ in range(5):
        assert torch.equal(spec_sample(t, d, drafts, u), out)


def test_draws_beside_a_border_of_nearly_equal_distributions():
    """Draft and target differ by a millionth (the draft's logits all higher by
    some amount, which changes nothing), so that p - q cancels all but the last
    third of a double: weights good to 2^-47 leave the border between two tokens
    of the residual within 4e-8 of its place in u (2^-47 of a weight over a
    residual of at least 2e-7 of it), and 2.5e-7 beside it (two to four steps of
    u) the pick is decided."""
    B = 8192
    g = torch.Generator(device="cuda")
    g.manual_seed(12)
    t = 2.0 * torch.randn((2, B, 3), generator=g, device="cuda")
    d = t[:1] + 4.0 * torch.rand((1, B, 1), generator=g, device="cuda")
    d[..., 2] += 4e-6  # the draft's token, a hair likelier than in the target: rejected by u_0, residual on 0 and 1
    p, q = torch.softmax(t[0].double(), 1), torch.softmax(d[0].double(), 1)
    r = (p - q)[:, :2]
    top = 1.0 - 2.0 ** -24
    use = (r > 2e-7 * p[:, :2]).all(1) & (top * q[:, 2] >= p[:, 2] * (1 + 1e-9))
    border = r[:, 0] / r.sum(1)
    use &= (border > 0.01) & (border < 0.99)
    assert use.sum() > 1000
    side = torch.arange(B, device="cuda") % 2  # below or above the border
    u = torch.stack([torch.full((B,), top, dtype=torch.float64, device="cuda"), border + (side * 2 - 1) * 2.5e-7], 1).float()
    drafts = torch.full((B, 1), 2, dtype=torch.int32, device="cuda")
    got = spec_sample(t, d, drafts, u)
    wg.context().sync()
    assert torch.equal(got[0][use].long(), side[use])


def test_hidden_logits_have_no_weight_at_any_maximum():
    """-inf beside one token, at every size of its logit and down to the lowest
    temperatures: that token is drawn."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    B, V = 2000, 70
    top = (torch.rand(B, generator=g, device="cuda") * 2 - 1) * 5000
    top[0] = 4897.20654
    at = torch.randint(0, V, (B,), generator=g, device="cuda")
    t = torch.full((1, B, V), -float("inf"), device="cuda")
    t[0, torch.arange(B, device="cuda"), at] = top
    for T in (1e-4, 0.001, 0.37, 1.0):
        u = torch.rand((B, 1), generator=g, device="cuda")
        got = spec_sample(t, None, None, u, temperature=T)
        wg.context().sync()
        assert torch.equal(got[0].long(), at)


def test_unaligned_rows_and_views():
    """Logits that start at any float (an odd vocabulary, a view)."""
    for off in range(4):
        g = torch.Generator(device="cuda")
        g.manual_seed(off)
        V = 8193
        flat = torch.randn(2 * V + off, generator=g, device="cuda")[off:]
        t = flat.view(1, 2, V)
        u = torch.rand((2, 1), generator=g, device="cuda")
        assert torch.equal(spec_sample(t, None, None, u).cpu(), R.spec_picks(t, None, None, u, 1.0))


def test_accept_applies_the_picks():
    """wg_spec_sample then wg_spec_accept keeps exactly the kept tokens and the
    drawn one."""
    B, k, V = 12, 4, 5000
    t, d, drafts, u = make(B, k, V, 0.6, seed=8)
    picks = spec_sample(t, d, drafts, u)
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    pos_t, pos_d, nt, nd, out, n, acc = z(B) + 105, z(B) + 105, z(B), z(B), z(B, 16), z(B), z(B)
    c = wg.context()
    c._check(_lib.lib().wg_spec_accept(c.handle, *[ctypes.c_void_p(x.data_ptr()) for x in (drafts, picks)], B, k,
                                       *[ctypes.c_void_p(x.data_ptr()) for x in (pos_t, pos_d, nt, nd, out)], 16,
                                       *[ctypes.c_void_p(x.data_ptr()) for x in (n, acc)]))
    c.sync()
    kept = (picks >= 0).sum(0).to(torch.int32)
    assert torch.equal(n, kept) and torch.equal(acc, kept - 1)
    for b in range(B):
        assert torch.equal(out[b, :kept[b]], picks[:kept[b], b])
    assert torch.equal(pos_t, 100 + kept) and torch.equal(nt, picks[kept.long() - 1, torch.arange(B)])


def test_graph_and_stream():
    t, d, drafts, u = make(4, 3, 20000, 0.5, seed=6)
    want = spec_sample(t, d, drafts, u)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        spec_sample(t, d, drafts, u, out=out)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    u.uniform_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), R.spec_picks(t, d, drafts, u, 1.0))


def test_the_draws_follow_the_target():
    """Over many sequences with equal rows, the first token's frequencies are
    the target's (drafts of another distribution): within 5 standard errors."""
    B, V = 20000, 6
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    row_t = torch.randn(V, generator=g, device="cuda")
    row_d = torch.randn(V, generator=g, device="cuda")
    t, d = row_t.expand(2, B, V).contiguous(), row_d.expand(1, B, V).contiguous()
    drafts = torch.multinomial(torch.softmax(row_d, 0), B, True, generator=g).to(torch.int32).view(B, 1)
    u = torch.rand((B, 2), generator=g, device="cuda")
    first = spec_sample(t, d, drafts, u)[0]
    p = torch.softmax(row_t.double(), 0)
    freq = torch.bincount(first.long(), minlength=V).double() / B
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()


def test_refusals():
    t, d, drafts, u = make(2, 1, 8, 0.5)
    S, A = wg.ShapeError, wg.GpuError
    for err, args in [(S, (t, None, None, u)), (S, (t, d, None, u)), (S, (t, d[:, :, :7], drafts, u)),
                      (S, (t, d, drafts, u[:, :1])), (A, (t.double(), d, drafts, u)), (A, (t, d, drafts.long(), u)),
                      (A, (t, d, drafts, u.cpu())), (S, (t.cpu(), d, drafts, u))]:
        with pytest.raises(err):
            spec_sample(*args)
    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-5):
        with pytest.raises(A):
            spec_sample(t, d, drafts, u, temperature=T)
    c, L = wg.context(), _lib.lib()
    x, n = t.data_ptr(), ctypes.c_size_t()

    def call(target=x, draft=x, drafts=x, batch=1, k=1, V=8, ws=x, ws_bytes=1 << 20):
        return L.wg_spec_sample(c.handle, target, draft, drafts, batch, k, V, 1.0, x, x, ws, ws_bytes)

    I, A, U = _lib.WG_INVALID_SHAPE, _lib.WG_INVALID_ARGUMENT, _lib.WG_UNSUPPORTED
    for st, kw in [(I, dict(k=33)), (I, dict(k=-1)), (I, dict(V=0)), (I, dict(V=(1 << 21) + 1)), (I, dict(batch=-1)),
                   (U, dict(batch=30000)), (A, dict(draft=None)), (A, dict(drafts=None)), (A, dict(target=x + 2)),
                   (A, dict(ws=None)), (A, dict(ws=x + 4)), (A, dict(ws_bytes=23)), (0, dict(batch=0))]:
        assert call(**kw) == st, kw
    assert L.wg_spec_sample_workspace(c.handle, 1, 1, 8, ctypes.byref(n)) == 0 and n.value == 24
    assert L.wg_spec_sample_workspace(c.handle, 1, 40, 8, ctypes.byref(n)) == I


def test_overlapping_tensors_are_refused():
    """picks and the workspace share no memory with the inputs or each other
    (nothing is launched)."""
    c, L = wg.context(), _lib.lib()
    c.use_torch_stream()
    B, k, V = 2, 1, 8
    x = torch.zeros(4096, device="cuda").data_ptr()
    at = dict(target=x, draft=x + 128, drafts=x + 192, u=x + 256, picks=x + 512, ws=x + 1024)
    size = dict(target=128, draft=64, drafts=8, u=16, picks=16, ws=48)

    def call(**kw):
        a = {**at, **kw}
        return L.wg_spec_sample(c.handle, a["target"], a["draft"], a["drafts"], B, k, V, 1.0, a["u"], a["picks"], a["ws"],
                                1024)

    A = _lib.WG_INVALID_ARGUMENT
    for what in ("target", "draft", "drafts", "u", "ws"):
        for p in (at[what], at[what] + size[what] - 4, at[what] - 12):
            assert call(picks=p) == A and "overlap" in L.wg_last_error(c.handle).decode(), what
    for what in ("target", "draft", "drafts", "u", "picks"):
        for p in (at[what], at[what] + size[what] - 8, at[what] - 40):
            assert call(ws=p) == A and "overlap" in L.wg_last_error(c.handle).decode(), what
    assert call() == 0 and call(picks=x + 272) == 0
    c.sync()
