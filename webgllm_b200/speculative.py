"""Speculative decoding, greedy or sampled (for the 8B shape: a 1.1B draft with
the 1.1B model's layout and the target's vocabulary proposes k = 4 tokens per
step).

The reference drafts on the host and verifies with forwardDraft / accept
(packages/webgllm/src/engine.ts:8035,8063). Here one step stays on the GPU
and is captured as one CUDA graph: the draft decodes k + 1 tokens (its own
greedy picks, from the last kept token; the extra step puts d_k in its cache
for when every proposal is kept), the target reads the last kept token and
d_1..d_k as k + 1 rows per sequence and picks after every row, and
wg_spec_accept keeps the longest agreeing prefix plus the target's own next
token, rewinding both models' positions (the KV caches are indexed by
position, so nothing else is undone there); models with gated short-conv
layers (config 3's hybrid) keep their conv state after every draft token
(wg_short_conv_prefixes) and set it back to the kept prefix's
(wg_conv_restore). Every emitted token is the target's greedy pick for
its position as the verify batch computes it, whatever the draft proposes.
A verify batch of more than 16 rows (batch x (k + 1)) runs on the
tensor-core GEMM, whose accumulation order (and fp16 weights) differ from
the decode GEMV's: its logits differ from a plain decode step's at the level
that any change of accumulation order produces in these models (~1e-3
relative, from activations that land on the other side of an fp16
rounding), so a near tie can be picked otherwise than plain greedy decoding
picks it (WG_OPT_EXACT_ROWS routes the verify through the GEMV: fewer such
ties, a slower round).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .model import DecoderConfig, DecoderModel
from .q4 import context_of, host_calls


def draft_config(target: DecoderConfig) -> DecoderConfig:
    """Config 2's layout with the target's vocabulary."""
    return DecoderConfig("draft-1.1b", 22, 2048, 32, 4, 64, 5632, target.vocab, 1e-5, 1e4)


def spec_sample(target: torch.Tensor, draft: torch.Tensor | None, drafts: torch.Tensor | None, u: torch.Tensor, *,
                temperature: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """wg_spec_sample: verifies drafts int32 [batch][k] by the logits target
    float32 [k + 1][batch][V] and draft float32 [k][batch][V] with the random
    numbers u float32 [batch][k + 1]. Returns picks int32 [k + 1][batch]: the
    kept tokens, then the drawn one, then -1 (what wg_spec_accept takes).
    draft and drafts None (k = 0): one token per sequence drawn from target
    [1][batch][V] (or [batch][V])."""
    host = host_calls()
    if host is not None:
        done = host.spec_sample(target, draft, drafts, u, temperature, out)
        if done is not None:
            return done
    if target.dim() == 2 and draft is None:
        target = target.unsqueeze(0)
    device = target.get_device()
    if target.dim() != 3 or device < 0:
        raise _lib.ShapeError(_lib.WG_INVALID_SHAPE, f"target {tuple(target.shape)} must be CUDA logits [k + 1][batch][V]")
    rows, batch, V = target.shape
    k = rows - 1
    if (draft is None) != (k == 0) or (drafts is None) != (k == 0):
        raise _lib.ShapeError(_lib.WG_INVALID_SHAPE, f"{k} drafted tokens a sequence need their draft logits and drafts")
    want = [(target, torch.float32, (rows, batch, V), "target"), (u, torch.float32, (batch, rows), "u")]
    if k:
        want += [(draft, torch.float32, (k, batch, V), "draft"), (drafts, torch.int32, (batch, k), "drafts")]
    if out is None:
        out = torch.empty((rows, batch), dtype=torch.int32, device=target.device)
    else:
        want.append((out, torch.int32, (rows, batch), "out"))
    for t, dt, shape, what in want:
        if t.shape != shape:
            raise _lib.ShapeError(_lib.WG_INVALID_SHAPE, f"{what} {tuple(t.shape)} must be {shape}")
        if t.dtype is not dt or t.get_device() != device or not t.is_contiguous():
            raise _lib.GpuError(_lib.WG_INVALID_ARGUMENT, f"{what} must be contiguous {dt} on CUDA device {device}")
    ctx, L = context_of(device), _lib.lib()
    need = ctypes.c_size_t()
    with ctx.lock:
        ctx._check(L.wg_spec_sample_workspace(ctx.handle, batch, k, V, ctypes.byref(need)))
    # from torch's allocator: safe on any stream and inside a graph
    ws = torch.empty(max(need.value, 8), dtype=torch.uint8, device=target.device)
    ctx.enqueue(L.wg_spec_sample, target.data_ptr(), draft.data_ptr() if k else None, drafts.data_ptr() if k else None,
                batch, k, V, temperature, u.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.nbytes)
    return out


class SpeculativeDecoder:
    """temperature 0: greedy, as above. temperature > 0: the draft's tokens are
    drawn from its own probabilities, kept against the target's, and the first
    that is not kept is drawn again from what the target has left
    (wg_spec_sample), so the emitted tokens are samples of the target whatever
    the draft proposes. step() uses the random numbers u and u_draft as they
    stand; run_step() has torch's generator of `seed` draw new ones before it."""

    def __init__(self, target: DecoderModel, draft: DecoderModel, k: int = 4, max_new: int = 512,
                 temperature: float = 0.0, seed: int = 0):
        if target.batch != draft.batch or target.cfg.vocab != draft.cfg.vocab:
            raise ValueError("target and draft must share batch and vocabulary")
        if target.max_rows < target.batch * (k + 1):
            raise ValueError(f"the target needs max_rows >= {target.batch * (k + 1)}")
        self.t, self.d, self.k = target, draft, k
        B = target.batch
        self.drafts = torch.zeros((B, max(k, 1)), dtype=torch.int32, device="cuda")
        self.picks = torch.zeros((k + 1, B), dtype=torch.int32, device="cuda")
        self.ver = torch.zeros((B, k + 1), dtype=torch.int32, device="cuda")
        self.out = torch.zeros((B, max_new + k + 1), dtype=torch.int32, device="cuda")
        self.out_len = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.accepted = torch.zeros(B, dtype=torch.int32, device="cuda")
        # conv models roll their state back to the kept prefix (convPrefixes /
        # accept, src/gpu/kernels.ts:1504, src/engine.ts:8063): positions
        # before the round, and the state after each of the k + 1 draft tokens
        self.pos_t0 = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.pos_d0 = torch.zeros(B, dtype=torch.int32, device="cuda")
        target.keep_prefixes(k + 1)
        draft.keep_prefixes(k + 1)
        self.graph = None
        self.temperature = temperature
        if temperature:
            if target.world > 1 or draft.world > 1:
                raise ValueError("sampled speculation needs the whole vocabulary on one GPU")
            V = target.cfg.vocab
            self.gen = torch.Generator(device="cuda")
            self.gen.manual_seed(seed)
            self.t_logits = torch.zeros((k + 1, B, V), device="cuda")
            self.d_logits = torch.zeros((max(k, 1), B, V), device="cuda")
            self.u = torch.zeros((B, k + 1), device="cuda")
            self.u_draft = torch.zeros((max(k, 1), B, 1), device="cuda")

    def prefill(self, prompts: torch.Tensor):
        """Both models read the prompts; the first emitted token is the
        target's pick."""
        self.t.prefill(prompts)
        self.d.prefill(prompts)
        self.out_len.zero_()
        self.accepted.zero_()
        if self.temperature:
            u = torch.rand((self.t.batch, 1), generator=self.gen, device="cuda")
            spec_sample(self.t.logits, None, None, u, temperature=self.temperature, out=self.t.next_id.view(1, -1))
        self.out[:, 0].copy_(self.t.next_id)
        self.out_len.fill_(1)
        self.d.next_id.copy_(self.t.next_id)
        self.draw()

    def step(self):
        """One draft-and-verify round (every sequence gains 1 .. k + 1 tokens)."""
        t, d, k = self.t, self.d, self.k
        self.ver[:, 0].copy_(t.next_id)
        if d.has_conv:
            self.pos_d0.copy_(d.pos)
        if t.has_conv:
            self.pos_t0.copy_(t.pos)
        for j in range(k + 1):
            d.prefix_slot = j if d.has_conv else None
            d.row_logits = self.d_logits[j:j + 1] if self.temperature and j < k else None
            try:
                d.decode_step()
            finally:
                d.prefix_slot = None
                d.row_logits = None
            if j < k:
                if self.temperature:
                    spec_sample(self.d_logits[j], None, None, self.u_draft[j], temperature=self.temperature,
                                out=d.next_id.view(1, -1))
                self.drafts[:, j].copy_(d.next_id)
                self.ver[:, j + 1].copy_(d.next_id)
        t.row_picks = self.picks
        t.row_logits = self.t_logits if self.temperature else None
        t.prefix_slot = 0 if t.has_conv else None
        try:
            t.forward(self.ver.reshape(-1), t.batch * (k + 1))
        finally:
            t.row_picks = None
            t.row_logits = None
            t.prefix_slot = None
        if self.temperature:
            spec_sample(self.t_logits, self.d_logits if k else None, self.drafts if k else None, self.u,
                        temperature=self.temperature, out=self.picks)
        t.ctx.enqueue(_lib.lib().wg_spec_accept, self.drafts.data_ptr(), self.picks.data_ptr(), t.batch, k,
                      t.pos.data_ptr(), d.pos.data_ptr(), t.next_id.data_ptr(), d.next_id.data_ptr(),
                      self.out.data_ptr(), self.out.shape[1], self.out_len.data_ptr(), self.accepted.data_ptr())
        t.restore_prefix(self.pos_t0)
        d.restore_prefix(self.pos_d0)

    def capture(self):
        """Records step() as one CUDA graph (after one eager step)."""
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.step()

    def draw(self):
        """New random numbers for the next round."""
        if self.temperature:
            self.u.uniform_(generator=self.gen)
            self.u_draft.uniform_(generator=self.gen)

    def run_step(self):
        self.draw()
        if self.graph is not None:
            self.graph.replay()
        else:
            self.step()
