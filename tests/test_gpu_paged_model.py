"""The paged cache and sampled speculation as a model uses them: a random-init
decoder whose keys and values live in pages, with and without a window, and
draft / verify / accept over it."""
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import decoder_reference as R  # noqa: E402
import paged_reference as PR  # noqa: E402
from webgllm_b200.model import DecoderConfig, DecoderModel  # noqa: E402
from webgllm_b200.paged import PagedCache  # noqa: E402
from webgllm_b200.speculative import SpeculativeDecoder, spec_sample  # noqa: E402

LLAMA = DecoderConfig("tiny-llama", 3, 256, 8, 2, 64, 768, 1000, 1e-5, 1e4)
HYBRID = DecoderConfig("tiny-hybrid", 4, 256, 8, 2, 64, 512, 1000, 1e-5, 1e6, ["conv", "attn", "conv", "attn"], 3, True)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def model(cfg, batch, length=128, page=16, spare=3, reserve=True, max_rows=64, **kw):
    """A paged model whose pages hold NaN until they are written."""
    n = sum(t == "attn" for t in cfg.layer_types)
    c = PagedCache(n, batch, cfg.kv_heads, cfg.head_dim, batch * (-(-length // page)) + spare, length, page_size=page)
    c.k.fill_(float("nan"))
    c.v.fill_(float("nan"))
    if reserve:
        for b in range(batch):
            c.reserve(b, length)
    return DecoderModel(cfg, batch=batch, max_rows=max_rows, cache=c, keep_blocks=True, **kw)


@pytest.mark.parametrize("cfg", [LLAMA, HYBRID], ids=lambda c: c.name)
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_paged_decoder_matches_reference_forward(cfg, window, sinks, monkeypatch):
    """Prefill 40 tokens of two sequences, then 6 steps (eager, then a graph's
    replays) against the torch fp32 forward: logits within 2 % of their scale,
    the bound of the contiguous caches' test."""
    if window:
        def attention(q, kc, vc, pos0, H, Hkv):
            rows = q.shape[0]
            L = pos0 + rows
            k, v = (t[:, :L].float().repeat_interleave(H // Hkv, 0) for t in (kc, vc))
            s = torch.einsum("rhd,hld->hrl", q.float().view(rows, H, -1), k)
            i = torch.arange(pos0, L, device="cuda")[:, None]
            see = PR.sees(i, torch.arange(L, device="cuda")[None], window, sinks)
            return torch.einsum("hrl,hld->rhd", torch.softmax(s.masked_fill(~see, -float("inf")), -1), v)

        monkeypatch.setattr(R, "attention", attention)
    m = model(cfg, 2, seed=3, window=window, sinks=sinks)
    refs = [R.ReferenceDecoder(m), R.ReferenceDecoder(m)]
    prompts = torch.randint(0, cfg.vocab, (2, 20), generator=gen(9), device="cuda").to(torch.int32)
    m.prefill(prompts)
    for step in range(7):
        for b in range(2):
            want = refs[b].forward(prompts[b] if step == 0 else tok[b:b + 1])  # noqa: F821
            assert (m.logits[b] - want).abs().max().item() < 2e-2 * want.abs().max().item(), (step, b)
        tok = m.next_id.clone()
        if step == 0:
            m.decode_step()
            m.capture_decode()
        else:
            m.graph.replay()
        m.ctx.sync()
    assert m.pos.tolist() == [27, 27]


def test_freed_pages_change_nothing():
    """A windowed model that gives its pages back as the window passes them
    emits the same bits as one that keeps them, from a pool that could not hold
    the whole sequence."""
    window, sinks, n = 32, 4, 90
    keep = model(LLAMA, 1, length=128, seed=5, window=window, sinks=sinks)
    tight = model(LLAMA, 1, length=128, seed=5, window=window, sinks=sinks, reserve=False, spare=0)
    del tight.cache.free[6:]  # 6 pages of 16 in all
    prompt = torch.randint(0, LLAMA.vocab, (1, 20), generator=gen(2), device="cuda").to(torch.int32)
    tight.cache.reserve(0, 20)
    for m in (keep, tight):
        m.prefill(prompt)
    assert torch.equal(keep.logits, tight.logits)
    freed = 0
    for i in range(n):
        pos = 20 + i
        freed += tight.cache.trim(0, pos, window, sinks)
        tight.cache.reserve(0, pos + 1, start=pos)
        keep.decode_step()
        tight.decode_step()
        assert torch.equal(keep.logits, tight.logits), i
    keep.ctx.sync()
    assert freed >= 3


def test_long_prompts_match_decode_steps():
    """A prompt read at once (tensor-core attention) and token by token: the
    keys and values in the pages agree to their rounding, the last logits to 2 %."""
    cfg = DecoderConfig("tiny-wide", 2, 512, 32, 8, 64, 512, 500, 1e-5, 1e4)
    prompt = torch.randint(0, cfg.vocab, (1, 200), generator=gen(3), device="cuda").to(torch.int32)
    a = model(cfg, 1, length=224, seed=1, max_rows=256, page=32)
    b = model(cfg, 1, length=224, seed=1, max_rows=256, page=32)
    a.prefill(prompt)
    for i in range(200):
        b.forward(prompt[0, i:i + 1].contiguous(), 1)
    a.ctx.sync()
    assert (a.logits - b.logits).abs().max().item() < 2e-2 * b.logits.abs().max().item()


@pytest.mark.parametrize("cfg", [LLAMA, HYBRID], ids=lambda c: c.name)
@pytest.mark.parametrize("k", [1, 4])
def test_sampled_speculation(cfg, k):
    """Rounds of draft, sample, verify, accept over paged caches, eager and
    replayed from a graph: each round's picks are the definition's for the
    logits and random numbers it used, and exactly those are emitted."""
    B, T = 3, 0.9
    t = model(cfg, B, seed=11)
    d = model(cfg, B, seed=11)
    d.final_norm.mul_(1.0 + 0.5 * torch.rand(cfg.hidden, generator=gen(15), device="cuda"))
    spec = SpeculativeDecoder(t, d, k=k, max_new=96, temperature=T, seed=4)
    prompts = torch.randint(0, cfg.vocab, (B, 12), generator=gen(21), device="cuda").to(torch.int32)
    spec.prefill(prompts)
    assert ((spec.out[:, 0] >= 0) & (spec.out[:, 0] < cfg.vocab)).all()
    kept = 0
    for i in range(8):
        before, pos = spec.out_len.clone(), t.pos.clone()
        spec.draw()
        if i == 0:
            spec.step()
        else:
            if i == 1:
                torch.cuda.synchronize()
                spec.capture()
            spec.graph.replay()
        t.ctx.sync()
        want = PR.spec_picks(spec.t_logits, spec.d_logits, spec.drafts, spec.u, T)
        assert torch.equal(spec.picks.cpu(), want), i
        # the draft's own tokens
        for j in range(k):
            own = PR.spec_picks(spec.d_logits[j:j + 1], None, None, spec.u_draft[j], T)
            assert torch.equal(spec.drafts[:, j].cpu(), own[0]), (i, j)
        n = (want >= 0).sum(0)
        assert torch.equal((spec.out_len - before).cpu(), n.to(torch.int32))
        assert torch.equal((t.pos - pos).cpu(), n.to(torch.int32)) and torch.equal(t.pos, d.pos)
        for b in range(B):
            assert torch.equal(spec.out[b, before[b]:spec.out_len[b]].cpu(), want[:n[b], b])
        kept += int((n - 1).sum())
    assert 0 < kept < 8 * B * k  # some drafts kept, some not


def test_low_temperature_is_greedy_speculation():
    """At a temperature where every draw is the maximum, sampled speculation
    emits the greedy tokens (the same verify arithmetic: equal picks)."""
    B, k = 2, 4
    prompts = torch.randint(0, LLAMA.vocab, (B, 16), generator=gen(2), device="cuda").to(torch.int32)
    outs = []
    for T in (0.0, 1e-4):
        t, d = model(LLAMA, B, seed=7), model(LLAMA, B, seed=8)
        spec = SpeculativeDecoder(t, d, k=k, max_new=64, temperature=T)
        spec.prefill(prompts)
        for _ in range(10):
            spec.run_step()
        torch.cuda.synchronize()
        outs.append(spec.out[:, :11].clone())
    # (a gap of logits below 1e-4 x 30 could be drawn either way: none here)
    assert torch.equal(outs[0], outs[1])


def test_a_model_and_calls_from_another_thread():
    """Decode steps on one thread's stream while another thread samples and
    attends on its own: each call's launches stay on its thread's stream."""
    m = model(LLAMA, 2, seed=3)
    prompts = torch.randint(0, LLAMA.vocab, (2, 20), generator=gen(9), device="cuda").to(torch.int32)

    def steps(n=40):
        m.reset()
        m.prefill(prompts)
        logits = []
        for _ in range(n):
            m.decode_step()
            logits.append(m.logits.clone())
        return torch.stack(logits)

    rows, u = torch.randn((8, 32000), generator=gen(4), device="cuda"), torch.rand((8, 1), generator=gen(5), device="cuda")
    want, picks = steps(), spec_sample(rows, None, None, u)
    torch.cuda.synchronize()
    wrong, stop = [], threading.Event()

    def other():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            while not stop.is_set():
                mine = rows.clone()
                got = spec_sample(mine, None, None, u)
                mine.fill_(float("nan"))
                s.synchronize()
                if not torch.equal(got, picks):
                    wrong.append(got)

    t = threading.Thread(target=other)
    t.start()
    try:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got = steps()
                s.synchronize()
                assert torch.equal(got, want)
    finally:
        stop.set()
        t.join()
    assert not wrong
    torch.cuda.synchronize()
    m.ctx.sync()


def test_model_refusals():
    c = PagedCache(2, 1, 2, 64, 4, 64, page_size=16)
    with pytest.raises(ValueError):
        DecoderModel(LLAMA, cache=c)  # three attention layers
    with pytest.raises(ValueError):
        DecoderModel(LLAMA, window=16)
