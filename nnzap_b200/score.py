"""Scoring and continuing many prompts at once over one paged KV cache.

The reference prefills one prompt token by token into its one contiguous cache
and samples from host logits (nnmetal/src/transformer.zig:4032-4123,
:3694-3880).  Here any number of sequences share a pool of K/V pages, and each
step runs a ragged batch of their tokens -- pieces of prompts and single new
tokens alike -- through the ragged-serving operators of :mod:`nnzap_b200.paged`
(norm + rotation into pages, attention over pages, log probabilities) and the
quantized GEMM of the library; the glue between them is elementwise torch.

    python -m nnzap_b200.score --tokens 700,33,1,512 --new 8 [--budget 512] [--layers 28]

builds the Bonsai-1.7B architecture with seeded random 1-bit weights, scores
seeded random prompts of those lengths and continues each greedily.
"""
from __future__ import annotations

import argparse
import dataclasses
import time

import numpy as np
import torch

from . import _capi as capi
from . import paged
from ._capi import check, lib
from .engine import TransformerConfig


class _Weights:
    """One quantized matrix [M][K] in the reference's flat layout, on the device."""

    def __init__(self, cfg: TransformerConfig, parts: list, K: int, device):
        q1 = cfg.quant_format == "q1_0"
        self.fmt, self.K, self.gs = (capi.NNZ_Q1 if q1 else capi.NNZ_Q4), K, cfg.group_size
        self.scale_dtype = capi.NNZ_SCALE_BF16 if not q1 and cfg.scale_dtype == "bf16" else capi.NNZ_SCALE_F16

        def dev(key, as_dtype):    # rows of several matrices one after the other
            return torch.from_numpy(np.concatenate([np.ascontiguousarray(p[key]).view(np.uint8).reshape(-1) for p in parts])
                                    .view(as_dtype)).to(device)
        self.w = dev("weight", np.uint8)
        self.s = dev("scales", np.int16)
        if q1 and cfg.q1_scales_are_mlx:
            self.s = (self.s.view(torch.float16) / 2).view(torch.int16)
        self.b = None if q1 else dev("biases", np.int16)
        self.M = self.w.numel() * (8 if q1 else 2) // K

    def gemm(self, x: torch.Tensor, out: torch.Tensor | None = None, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """x [T][K] float16 times the transpose: float16 or float32 [T][M], or added to float32 ``out``."""
        kind = capi.NNZ_OUT_F32_ADD
        if out is None:
            kind = capi.NNZ_OUT_F16 if dtype is torch.float16 else capi.NNZ_OUT_F32
            out = torch.empty(x.shape[0], self.M, dtype=dtype, device=x.device)
        check(lib().nnz_prefill_gemm(self.fmt, self.scale_dtype, self.w.data_ptr(), self.s.data_ptr(),
                                     None if self.b is None else self.b.data_ptr(), x.shape[0], self.K, self.M, self.gs,
                                     x.data_ptr(), out.data_ptr(), kind, paged._stream(x.device.index)))
        return out

    def rows(self, ids: torch.Tensor) -> torch.Tensor:
        """Dequantized rows, float32 [len(ids)][K] (the embedding lookup); NaN for an id that is none (indexing with it
        would stop the device)."""
        none = (ids < 0) | (ids >= self.M)
        return torch.where(none[:, None], torch.nan, self._rows(torch.where(none, 0, ids)))

    def _rows(self, ids: torch.Tensor) -> torch.Tensor:
        g = self.s.view(self.M, self.K // self.gs)[ids].view(torch.bfloat16 if self.scale_dtype else torch.float16).float()
        if self.fmt == capi.NNZ_Q1:
            bits = self.w.view(self.M, self.K // 8)[ids]
            sign = ((bits[..., None] >> torch.arange(8, device=ids.device, dtype=torch.uint8)) & 1).view(len(ids), -1, self.gs).float() * 2 - 1
            return (sign * g[..., None]).view(len(ids), self.K)
        bias = self.b.view(self.M, self.K // self.gs)[ids].view(torch.bfloat16 if self.scale_dtype else torch.float16).float()
        byte = self.w.view(self.M, self.K // 2)[ids]
        q = torch.stack([byte & 15, byte >> 4], -1).view(len(ids), -1, self.gs).float()
        return (q * g[..., None] + bias[..., None]).view(len(ids), self.K)


class PagedModel:
    """The quantized Qwen3 decoder over a paged KV cache: ``step`` runs the new
    tokens of any number of sequences."""

    def __init__(self, config: TransformerConfig, tensors, num_pages: int, page_size: int = 16, device="cuda"):
        """``tensors``: (checkpoint name, array) pairs as ``Model.load_weights`` takes them."""
        c, t = config, dict(tensors)
        device = torch.device(device)
        self.config, self.device = c, torch.device("cuda", torch.cuda.current_device()) if device.index is None else device
        H, hd = c.hidden_size, c.head_dim

        def q(*names):
            keys = ("weight", "scales") + (("biases",) if c.quant_format == "q4_mlx" else ())
            return [{k: t[f"{n}.{k}"] for k in keys} for n in names]

        def f32(name):
            return torch.from_numpy(np.ascontiguousarray(t[name], dtype=np.float32)).to(self.device)
        self.embed = _Weights(c, q("model.embed_tokens"), H, self.device)
        self.lm_head = self.embed if c.tie_word_embeddings else _Weights(c, q("lm_head"), H, self.device)
        self.final_norm = f32("model.norm.weight")
        self.table = paged.rope_table(c.rope_theta, hd, c.max_context_length, self.device)
        self.layers, workspace = [], None
        for i in range(c.num_layers):
            p = f"model.layers.{i}."
            kv = paged.PagedKV.empty(num_pages, c.num_kv_heads, page_size, hd, device=self.device)
            self.layers.append({
                "kv": kv, "attn_norm": f32(p + "input_layernorm.weight"), "ffn_norm": f32(p + "post_attention_layernorm.weight"),
                "qkv": _Weights(c, q(p + "self_attn.q_proj", p + "self_attn.k_proj", p + "self_attn.v_proj"), H, self.device),
                "o": _Weights(c, q(p + "self_attn.o_proj"), c.query_dim, self.device),
                "gate": _Weights(c, q(p + "mlp.gate_proj"), H, self.device), "up": _Weights(c, q(p + "mlp.up_proj"), H, self.device),
                "down": _Weights(c, q(p + "mlp.down_proj"), c.intermediate_size, self.device),
                "write": paged.QKNormRope(kv, c.num_query_heads, f32(p + "self_attn.q_norm.weight"), f32(p + "self_attn.k_norm.weight"),
                                          self.table, eps=c.eps, rope_style=c.rope_style),
                "attend": paged.PagedAttention(kv, c.num_query_heads, workspace=workspace)})      # layers run one after the other
            workspace = self.layers[-1]["attend"].workspace
        self.free = list(range(num_pages))[::-1]
        self.page_size = page_size

    def _norm(self, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.config.eps) * w).half()

    def step(self, tokens, positions, slots, page_table, q_start, kv_len, max_new: int) -> torch.Tensor:
        """float32 logits [len(tokens)][vocab]; device tensors as the operators take them."""
        if paged._current_device() != self.device.index:      # the GEMMs run on the current device
            with paged._device(self.device.index):
                return self.step(tokens, positions, slots, page_table, q_start, kv_len, max_new)
        x = self.embed.rows(tokens.long())
        for L in self.layers:
            qkv = L["qkv"].gemm(self._norm(x, L["attn_norm"]))
            q = L["write"](qkv, positions, slots)
            a = L["attend"](q, page_table, q_start, kv_len, max_new)
            L["o"].gemm(a, out=x)
            h = self._norm(x, L["ffn_norm"])
            g, u = L["gate"].gemm(h).float(), L["up"].gemm(h).float()
            L["down"].gemm((g * torch.sigmoid(g) * u).half(), out=x)
        return self.lm_head.gemm(self._norm(x, self.final_norm), dtype=torch.float32)


@dataclasses.dataclass
class Scored:
    """One sequence: its prompt, then what was generated."""
    tokens: list
    logprobs: list            # of tokens[1:], each given those before it
    entropies: list           # of the same distributions
    top_ids: list             # their most probable tokens, in order
    top_logprobs: list


def score(model: PagedModel, prompts, new_tokens: int = 0, budget: int = 512, top_k: int = 5) -> list:
    """Log probability, entropy and alternatives of every prompt token, and of
    ``new_tokens`` greedily generated ones; at most ``budget`` tokens a step,
    taken from the sequences in turn as far as there are pages.  A sequence's
    pages are free again when it is done; MemoryError if none can go on."""
    dev, page = model.device, model.page_size
    seqs = [Scored([int(t) for t in p], [], [], [], []) for p in prompts]
    cfg = model.config
    paged._need(new_tokens >= 0 and budget > 0 and 1 <= top_k <= 32, "score: new_tokens >= 0, budget > 0, top_k 1 .. 32")
    for i, s in enumerate(seqs):
        paged._need(len(s.tokens) > 0, f"prompt {i} is empty")
        paged._need(all(0 <= t < cfg.vocab_size for t in s.tokens), f"prompt {i} has a token outside 0 .. {cfg.vocab_size - 1}")
        paged._need(len(s.tokens) + new_tokens - 1 <= cfg.max_context_length,
                    f"prompt {i}: {len(s.tokens)} and {new_tokens} new tokens do not fit a context of {cfg.max_context_length}")
    goal = [len(s.tokens) + new_tokens for s in seqs]
    pages = [[] for _ in seqs]
    done = [0] * len(seqs)                       # tokens whose keys are in the cache
    try:
        while True:
            # what each sequence contributes: tokens that are known and not yet run,
            # whose successor is still wanted, and that pages can be had for
            left, take = budget, []
            for i, s in enumerate(seqs):
                n = min(left, min(len(s.tokens), goal[i] - 1) - done[i], (len(pages[i]) + len(model.free)) * page - done[i])
                if n > 0:
                    take.append((i, n))
                    left -= n
                    while len(pages[i]) * page < done[i] + n:
                        pages[i].append(model.free.pop())
            if not take:
                if any(d < g - 1 for d, g in zip(done, goal)):
                    raise MemoryError("no free pages")
                return seqs
            tok, pos, slot, nxt = [], [], [], []
            for i, n in take:
                for p in range(done[i], done[i] + n):
                    tok.append(seqs[i].tokens[p])
                    pos.append(p)
                    slot.append(pages[i][p // page] * page + p % page)
                    nxt.append(seqs[i].tokens[p + 1] if p + 1 < len(seqs[i].tokens) else -1)
            width = max(len(pages[i]) for i, _ in take)
            i32 = dict(dtype=torch.int32, device=dev)
            logits = model.step(torch.tensor(tok, **i32), torch.tensor(pos, **i32), torch.tensor(slot, dtype=torch.int64, device=dev),
                                torch.tensor([pages[i] + [-1] * (width - len(pages[i])) for i, _ in take], **i32),
                                torch.tensor(np.cumsum([0] + [n for _, n in take]), **i32),
                                torch.tensor([done[i] + n for i, n in take], **i32), max(n for _, n in take))
            r = paged.token_logprobs(logits, torch.tensor(nxt, **i32), top_k=top_k)
            lp, ent, ids, top = (x.cpu().tolist() for x in (r.logprob, r.entropy, r.top_ids, r.top_logprobs))
            paged.stream_check(dev)
            row = 0
            for i, n in take:
                s = seqs[i]
                for _ in range(n):
                    done[i] += 1
                    if nxt[row] < 0:               # generate: the most probable token
                        if ids[row][0] < 0:
                            raise RuntimeError(f"prompt {i}: no token to continue with after {len(s.tokens)} (no logit is a number, or nothing is allowed)")
                        s.tokens.append(ids[row][0])
                        lp[row] = top[row][0]
                    s.logprobs.append(lp[row])
                    s.entropies.append(ent[row])
                    s.top_ids.append(ids[row])
                    s.top_logprobs.append(top[row])
                    row += 1
                if done[i] == goal[i] - 1:         # nothing of it is read again
                    model.free.extend(pages[i])
                    pages[i] = []
    finally:
        for p in pages:
            model.free.extend(p)


def main():
    from . import config_from_dims, synth
    ap = argparse.ArgumentParser(prog="python -m nnzap_b200.score")
    ap.add_argument("--tokens", default="700,33,1,512", help="prompt lengths")
    ap.add_argument("--new", type=int, default=8, help="tokens to generate for each")
    ap.add_argument("--budget", type=int, default=512, help="most tokens a step")
    ap.add_argument("--layers", type=int, default=28)
    ap.add_argument("--top-k", type=int, default=5)
    args = ap.parse_args()
    lens = [int(n) for n in args.tokens.split(",")]
    d = dataclasses.replace(synth.BONSAI_1_7B_Q1, layers=args.layers)
    W = synth.make_model(d, seed=0)
    page = 16
    m = PagedModel(config_from_dims(d, max_context_length=max(lens) + args.new + 1), synth.iter_named_tensors(W),
                   num_pages=sum(-(-(n + args.new) // page) for n in lens), page_size=page)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, d.vocab, n) for n in lens]
    score(m, [p[:2] for p in prompts])            # first launches
    t0 = time.perf_counter()
    out = score(m, prompts, new_tokens=args.new, budget=args.budget, top_k=args.top_k)
    dt = time.perf_counter() - t0
    for n, s in zip(lens, out):
        nll = -np.mean(s.logprobs[:n - 1]) if n > 1 else float("nan")
        print(f"prompt of {n}: mean -log p {nll:.3f}, mean entropy {np.mean(s.entropies):.3f}, continued with {s.tokens[n:]}")
    print(f"{sum(len(s.tokens) for s in out)} tokens in {dt * 1e3:.1f} ms")


if __name__ == "__main__":
    main()
