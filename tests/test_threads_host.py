"""Callers on several threads share a device's context (no GPU: a library that
records its calls): a stream choice and the calls that go with it are one step."""
import threading
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from webgllm_b200 import _lib, q4  # noqa: E402
from webgllm_b200.model import DecoderModel  # noqa: E402
from webgllm_b200.speculative import SpeculativeDecoder  # noqa: E402


@pytest.fixture
def recorded(monkeypatch):
    """(context, calls): each library call with whether the context's lock was held."""
    ctx = object.__new__(q4.Context)
    ctx.device, ctx.handle, ctx.lock = 0, None, threading.Lock()
    calls = []

    class Library:
        def __getattr__(self, name):
            def call(*args):
                calls.append((name, ctx.lock.locked()))
                return 0

            return call

    library = Library()
    monkeypatch.setattr(_lib, "lib", lambda: library)
    monkeypatch.setattr(q4, "_current_device", lambda: 0)
    monkeypatch.setattr(q4, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=0))
    return ctx, calls


def held(calls, *names):
    assert [n for n, _ in calls] == list(names)
    assert all(locked for _, locked in calls)


def test_matmul_holds_the_stream(recorded):
    ctx, calls = recorded
    w = SimpleNamespace(K=32, N=4, ctx=ctx, handle=1)
    q4.matmul(torch.zeros(2, 32), w)
    held(calls, "wg_set_stream", "wg_q4_matmul")
    assert not ctx.lock.locked()


@pytest.mark.parametrize("fused", [True, False])
def test_forward_holds_the_stream(recorded, fused):
    ctx, calls = recorded
    m = object.__new__(DecoderModel)
    m.ctx, m.batch, m.max_rows, m.fused = ctx, 1, 4, fused
    m._forward_fused = m._forward_passes = lambda ids, rows: _lib.lib().wg_embed()
    m.forward(torch.zeros(2, dtype=torch.int32), 2)
    held(calls, "wg_embed")
    m._forward_fused = m._forward_passes = lambda ids, rows: 1 / 0
    with pytest.raises(ZeroDivisionError):
        m.forward(torch.zeros(2, dtype=torch.int32), 2)
    assert not ctx.lock.locked()


def test_restored_conv_states_hold_the_stream(recorded):
    ctx, calls = recorded
    m = object.__new__(DecoderModel)
    m.ctx, m.batch = ctx, 1
    m.cfg = SimpleNamespace(hidden=8, conv_width=3, layer_types=["conv"])
    m.layers = [{"type": "conv", "slot": 0}]
    m.conv_prefixes, m.conv_state, m.pos = torch.zeros(1, 1, 2, 2, 8), torch.zeros(1, 1, 2, 8), torch.zeros(1)
    m.restore_prefix(torch.zeros(1))
    held(calls, "wg_set_stream", "wg_conv_restore")


def test_speculative_accept_holds_the_stream(recorded):
    ctx, calls = recorded

    def model():
        return SimpleNamespace(ctx=ctx, batch=1, has_conv=False, next_id=torch.zeros(1, dtype=torch.int32),
                               pos=torch.zeros(1, dtype=torch.int32), decode_step=lambda: None,
                               forward=lambda ids, rows: None, restore_prefix=lambda pos: None,
                               _c=lambda status: _lib.check(status, ctx.handle))

    s = object.__new__(SpeculativeDecoder)
    s.t, s.d, s.k, s.temperature = model(), model(), 1, 0.0
    s.drafts, s.ver = torch.zeros((1, 1), dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    s.picks, s.out = torch.zeros((2, 1), dtype=torch.int32), torch.zeros((1, 8), dtype=torch.int32)
    s.out_len = s.accepted = s.pos_t0 = s.pos_d0 = torch.zeros(1, dtype=torch.int32)
    s.step()
    held(calls, "wg_set_stream", "wg_spec_accept")


def test_a_refusal_is_read_before_another_call(recorded, monkeypatch):
    """The context's last error belongs to the call that failed."""
    ctx, _ = recorded
    seen = []

    def check(status, handle=None):
        seen.append((status, ctx.lock.locked()))
        raise _lib.GpuError(status, "refused")

    monkeypatch.setattr(q4, "check", check)
    with pytest.raises(_lib.GpuError):
        ctx.enqueue(lambda handle: 7)
    assert seen == [(7, True)] and not ctx.lock.locked()
