"""The text decoder on a paged cache, assembled from the device operators.

`PagedDecoder` runs the decoder's layers (decoder.zig:165-287) for any mix of sequences in one step, prompt
chunks beside single tokens: norms, projections and SwiGLU through `qwc_op_*`, and per layer one
`paged.append` and one `paged.attention` on that layer's pool. `sampling.sample` draws the next tokens.
Sequences own pages, not slots: a forked sequence shares its full pages with its parent and copies only the
page that it goes on writing, so n transcripts of a clip hold the clip's positions once.

    python -m qwenscriber_b200.paged_decoder      # a small synthetic model: one prompt, four sampled transcripts

Torch holds the memory and moves it (gathers of embedding rows, page copies, residual sums); the engine with
its own slots and fused steps is `runtime.CudaModel`.
"""

from __future__ import annotations

import contextlib
import dataclasses

import numpy as np
import torch

from . import paged, quant, sampling, synthetic
from .runtime import check, lib, rope_tables

COLUMNS = 64  # rows of activations that one qwc_op_gemm_streams call takes


@dataclasses.dataclass
class Matrix:
    fmt: int
    rows: int
    cols: int
    scales: torch.Tensor
    codes: torch.Tensor


@dataclasses.dataclass
class Sequence:
    pages: list
    length: int = 0


class PagedDecoder:
    """A decoder's weights and its pools of pages on one device."""

    def __init__(self, model: synthetic.Model, pages: int, page_size: int, device="cuda:0"):
        c = self.config = model.config
        self.device, self.page_size = torch.device(device), page_size
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.weights = {}
        for t in model.tensors:
            if t.kind < synthetic.EMBED:
                continue  # the audio tower's
            self.weights[t.kind, t.layer] = self._matrix(t) if t.fmt != quant.F32 else self._put(
                np.ascontiguousarray(t.payload).view(np.float32).ravel())
        cos, sin = rope_tables(c.rope_theta, c.text_head_dim, c.max_positions)
        self.cos, self.sin = (self._put(a.reshape(c.max_positions, -1)) for a in (cos, sin))
        self.pools = [paged.PagedCache.zeros(pages, page_size, c.text_key_value_heads, c.text_head_dim, self.device)
                      for _ in range(c.text_layers)]
        self.holders = [0] * pages  # sequences that hold each page

    def _put(self, a: np.ndarray) -> torch.Tensor:
        return torch.from_numpy(np.ascontiguousarray(a)).to(self.device)

    def _matrix(self, t) -> Matrix:
        raw = self._put(np.ascontiguousarray(t.payload).view(np.uint8).ravel())
        s0, sn, c0, cn = quant.plane_layout(t.fmt, t.rows, t.cols)
        return Matrix(t.fmt, t.rows, t.cols, raw[s0:s0 + sn].clone(), raw[c0:c0 + cn].clone())

    # ---- pages ----

    def _take(self) -> int:
        for i, n in enumerate(self.holders):
            if n == 0:
                self.holders[i] = 1
                return i
        self._no_page()

    def _no_page(self):
        paged.refuse("limit_exceeded", "PagedDecoder: the pool has no free page")

    def start(self) -> Sequence:
        return Sequence([])

    def release(self, seq: Sequence) -> None:
        for p in seq.pages:
            self.holders[p] -= 1
        seq.pages, seq.length = [], 0

    def fork(self, seq: Sequence) -> Sequence:
        """A sequence with the same positions: full pages shared, the one in use copied."""
        full = seq.length // self.page_size
        if len(seq.pages) - full > self.holders.count(0):
            self._no_page()
        for p in seq.pages[:full]:
            self.holders[p] += 1
        out = Sequence(seq.pages[:full], seq.length)
        for p in seq.pages[full:]:
            new = self._take()
            for pool in self.pools:
                for plane in (pool.k_scales, pool.k_codes, pool.v_scales, pool.v_codes):
                    rows = plane.view(pool.pages, self.page_size, -1)
                    rows[new].copy_(rows[p])
            out.pages.append(new)
        return out

    # ---- operators ----

    def _call(self, name: str, *args) -> None:
        with paged.elsewhere(paged.cuda_index(self.device), name) or contextlib.nullcontext():
            check(getattr(lib(), name)(*args, paged.current_stream(self.device)), name)

    def _project(self, w: Matrix, x: torch.Tensor) -> torch.Tensor:
        out = torch.empty(x.shape[0], w.rows, dtype=torch.float32, device=self.device)
        for i in range(0, x.shape[0], COLUMNS):
            n = min(COLUMNS, x.shape[0] - i)
            self._call("qwc_op_gemm_streams", w.fmt, w.scales.data_ptr(), w.codes.data_ptr(), w.rows, w.cols, x[i].data_ptr(), n,
                       out[i].data_ptr())
        return out

    def _norm(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        out = torch.empty_like(x)
        self._call("qwc_op_rmsnorm", x.data_ptr(), weight.data_ptr(), x.shape[1], x.shape[0], self.config.text_rms_norm_eps,
                   out.data_ptr())
        return out

    def _embed(self, ids: torch.Tensor) -> torch.Tensor:
        e = self.weights[synthetic.EMBED, 0]
        scales, codes = e.scales.view(e.rows, -1)[ids].contiguous(), e.codes.view(e.rows, -1)[ids].contiguous()
        out = torch.empty(ids.numel(), e.cols, dtype=torch.float32, device=self.device)
        self._call("qwc_op_dequantize", e.fmt, scales.data_ptr(), codes.data_ptr(), ids.numel(), e.cols, out.data_ptr())
        return out

    # ---- steps ----

    def step(self, work: list[tuple[Sequence, np.ndarray, np.ndarray | None]]) -> torch.Tensor:
        """Runs each sequence's new tokens ids (where token_audio_pad stands, the next row of its audio rows)
        and returns the logits after the last of each, [sequences, vocab]. Waits for the device. A step that is
        refused, or fails, leaves every sequence as it was."""
        if not work:
            return torch.empty(0, self.config.vocab_size, dtype=torch.float32, device=self.device)
        self._check(work)
        before = [(seq, seq.length, len(seq.pages)) for seq, _, _ in work]
        try:
            for seq, ids, _ in work:
                seq.length += len(ids)
                while len(seq.pages) * self.page_size < seq.length:
                    seq.pages.append(self._take())
            logits = self._forward(work)
            paged.check_waits(device=self.device)
        except BaseException:
            for seq, length, count in before:
                for p in seq.pages[count:]:
                    self.holders[p] -= 1
                del seq.pages[count:]
                seq.length = length
            raise
        return logits

    def _check(self, work) -> None:
        """Refuses a step before anything of it is done."""
        c, call = self.config, "PagedDecoder.step"
        if len({id(seq) for seq, _, _ in work}) < len(work):
            paged.refuse("invalid_argument", call)
        pages = 0
        for seq, ids, audio in work:
            ids = np.asarray(ids)
            if ids.ndim != 1:
                paged.refuse("shape_mismatch", call)
            if ids.size == 0 or seq.length + ids.size > c.max_positions:
                paged.refuse("limit_exceeded", call)
            if ids.dtype.kind not in "iu" or ids.min() < 0 or ids.max() >= c.vocab_size:
                paged.refuse("invalid_argument", call)  # (an embedding row that is not there is an assertion on the device)
            if audio is not None and np.shape(audio) != (np.count_nonzero(ids == c.token_audio_pad), c.text_hidden_size):
                paged.refuse("shape_mismatch", call)
            pages += -(-(seq.length + ids.size) // self.page_size) - len(seq.pages)
        if pages > self.holders.count(0):
            self._no_page()

    def _forward(self, work) -> torch.Tensor:
        """The logits of a step whose sequences have their lengths and pages."""
        c = self.config
        lengths = [len(ids) for _, ids, _ in work]
        table = np.zeros((len(work), max(len(s.pages) for s, _, _ in work)), np.int32)
        for row, (seq, _, _) in zip(table, work):
            row[:len(seq.pages)] = seq.pages
        starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        context = np.asarray([s.length for s, _, _ in work], np.int32)
        batch = paged.PagedBatch(self._put(starts), self._put(context), self._put(table), tokens=int(starts[-1]),
                                 max_query=max(lengths), max_context=int(context.max()))
        ids = np.concatenate([np.asarray(i, np.int64) for _, i, _ in work])
        x = self._embed(self._put(ids))
        at = np.concatenate([int(o) + np.flatnonzero(np.asarray(i) == c.token_audio_pad)
                             for o, (_, i, a) in zip(starts, work) if a is not None] or [np.zeros(0, np.int64)])
        if at.size:
            x[self._put(at)] = self._put(np.concatenate([np.asarray(a, np.float32) for _, _, a in work if a is not None]))
        heads, dim = c.text_attention_heads, c.text_head_dim
        for layer in range(1, c.text_layers + 1):
            w = lambda kind: self.weights[kind, layer]  # noqa: E731, B023
            h = self._norm(x, w(synthetic.ATTN_NORM))
            q, k, v = (self._project(w(kind), h).unflatten(1, (-1, dim)) for kind in (synthetic.Q, synthetic.K, synthetic.V))
            pool = self.pools[layer - 1]
            paged.append(pool, batch, q, k, v, self.cos, self.sin, q_norm=w(synthetic.Q_NORM), k_norm=w(synthetic.K_NORM),
                         eps=c.text_rms_norm_eps, q_out=q)
            o = paged.attention(pool, batch, q)
            x = x + self._project(w(synthetic.O), o.view(-1, heads * dim))
            h = self._norm(x, w(synthetic.FFN_NORM))
            gate, up = self._project(w(synthetic.GATE), h), self._project(w(synthetic.UP), h)
            self._call("qwc_op_silu_mul", gate.data_ptr(), up.data_ptr(), gate.numel(), gate.data_ptr())
            x = x + self._project(w(synthetic.DOWN), gate)
        last = x[self._put(starts[1:].astype(np.int64) - 1)]
        head = self.weights[synthetic.EMBED if c.tied else synthetic.OUTPUT, 0]
        return self._project(head, self._norm(last, self.weights[synthetic.FINAL_NORM, 0]))

    def transcripts(self, prompt: synthetic.Prompt, count: int, max_tokens: int, generator: torch.Generator,
                    **settings) -> list[tuple[list[int], float]]:
        """`count` transcripts of one prompt, each with the sum of its tokens' log-probabilities. The prompt is run
        once; `settings` are sampling.sample's, one value for all."""
        c = self.config
        stop = {c.token_eos_primary, c.token_eos_secondary, c.token_endoftext}
        seqs = [self.start()]
        out, live = [([], 0.0) for _ in range(count)], list(range(count))
        try:
            logits = self.step([(seqs[0], prompt.tokens, prompt.audio)]).expand(count, -1).contiguous()
            for _ in range(count - 1):
                seqs.append(self.fork(seqs[0]))
            for _ in range(max_tokens):
                u = torch.rand(len(live), generator=generator).to(self.device)
                kinds = {k: torch.full((len(live),), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=self.device)
                         for k, v in settings.items()}
                tokens, logprobs = (t.tolist() for t in sampling.sample(logits, u, **kinds))
                for i, tok, lp in zip(live, tokens, logprobs):
                    out[i] = (out[i][0] + ([tok] if tok not in stop else []), out[i][1] + lp)
                going = [(i, tok) for i, tok in zip(live, tokens) if tok not in stop]
                live = [i for i, _ in going]
                if not live:
                    break
                logits = self.step([(seqs[i], np.asarray([tok]), None) for i, tok in going])
        finally:
            for s in seqs:
                self.release(s)
        return out


def main() -> None:
    config = dataclasses.replace(synthetic.qwen3_asr_0p6b(), text_layers=4, vocab_size=151936, max_positions=512)
    model = synthetic.make_model(config, quant.Q8, seed=3)
    decoder = PagedDecoder(model, pages=64, page_size=16)
    prompt = synthetic.make_prompt(config, 188, 8, seed=3)
    found = decoder.transcripts(prompt, 4, 24, torch.Generator().manual_seed(1), temperature=0.7, top_k=50, top_p=0.95)
    for tokens, score in sorted(found, key=lambda f: -f[1]):
        print(f"{score:9.3f}  {tokens}")
    print(f"pages held: {sum(n > 0 for n in decoder.holders)}")


if __name__ == "__main__":
    main()
