"""Batch-1 decode loop for a Llama-style decoder whose linears are packed
INT8-X layers, with the whole token step captured in one CUDA graph.

The reference drives HuggingFace `generate()` around its packed modules
(ixrun/generate.py:39-70, ixrun/engine.py:510-516) and records that whole-model
graph capture was not possible with HF's dynamic KV cache.  This runner keeps a
static KV cache and position tensors so that one token step is a fixed launch
sequence: per layer RMSNorm -> q/k/v packed GEMVs -> RoPE -> cache write ->
attention over the static cache -> o_proj GEMV -> RMSNorm -> gate/up GEMVs ->
SwiGLU -> down GEMV.  The packed linears run the fused decode+GEMV kernel; with
`glue="kernels"` the work between them is this library's glue kernels (residual
add + RMSNorm, RoPE + cache write, split-context attention, SwiGLU) and q|k|v
and gate|up are one fused packed tensor each: 9 launches per layer, all taking
part in programmatic dependent launch; with
`glue="eager"` it is plain torch.  A prompt (many rows) runs on the glue kernels too, with the
weights decoded and dense matmuls; eager torch with `glue="eager"` or a head_dim of 256.

`weights="packed"` uses StreamingLinear (fused kernels); `weights="decoded"`
builds the same model with the packed weights decoded to bf16 and dense
matmuls -- with eager glue the ground truth for greedy-token agreement.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from .engine import StreamingLinear
from .packed import DevicePacked


@dataclass
class LlamaConfig:
    n_layers: int = 24
    hidden: int = 2048
    intermediate: int = 6144
    n_heads: int = 16
    n_kv_heads: int = 8
    head_dim: int = 128
    vocab: int = 73448
    rope_theta: float = 10000.0
    rms_eps: float = 1e-5
    max_seq: int = 1280


LINEARS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def linear_shapes(cfg: LlamaConfig) -> dict:
    h, hd = cfg.hidden, cfg.head_dim
    return {
        "q_proj": (cfg.n_heads * hd, h), "k_proj": (cfg.n_kv_heads * hd, h), "v_proj": (cfg.n_kv_heads * hd, h),
        "o_proj": (h, cfg.n_heads * hd), "gate_proj": (cfg.intermediate, h), "up_proj": (cfg.intermediate, h),
        "down_proj": (h, cfg.intermediate),
    }


class _DenseLinear(torch.nn.Module):
    """bf16 weight decoded once from a packed dict (ground-truth path)."""

    def __init__(self, packed: dict):
        super().__init__()
        self.weight = DevicePacked(packed).decode(kind="bf16")

    def forward(self, x):
        return F.linear(x, self.weight)


def _rms(x, w, eps):
    v = x.float()
    return (v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * w


class FusedPackedLinear(torch.nn.Module):
    """Several packed linears that share their input (q|k|v, gate|up) as ONE resident tensor and one launch; every
    part keeps its own per-tensor scale (p6.P6Packed.fuse).  forward returns the parts' outputs."""

    def __init__(self, packed_parts: list):
        super().__init__()
        from .p6 import P6Packed

        self.res = P6Packed.fuse(packed_parts)
        self.in_features = self.res.in_f
        self._w_buf = None

    def _set_shared_buf(self, buf):
        self._w_buf = buf

    def forward(self, x):
        rows = x.numel() // self.in_features
        x2 = x.reshape(rows, self.in_features)
        if rows <= 8:
            y = self.res.gemv(x2)
        else:                                   # prefill: decode into the shared buffer, dense matmul
            y = F.linear(x2, self.res.decode(out=self._w_buf[: self.res.N], kind="bf16"))
        return [y[:, a:a + n] for a, n in self.res.sections]


class PackedLlama(torch.nn.Module):
    def __init__(self, cfg: LlamaConfig, packed_layers: list, embed: torch.Tensor, lm_head: torch.Tensor,
                 norms: list | None = None, weights: str = "packed", device="cuda", glue: str | None = None):
        """packed_layers[i][name] = packed dict of layer i's linear `name`;
        embed [vocab, hidden] and lm_head [vocab, hidden] stay bf16.
        glue: "kernels" (default for packed weights) or "eager" (default for decoded weights)."""
        super().__init__()
        if weights not in ("packed", "decoded"):
            raise ValueError("weights must be 'packed' or 'decoded'")
        glue = glue or ("kernels" if weights == "packed" else "eager")
        if glue not in ("kernels", "eager"):
            raise ValueError("glue must be 'kernels' or 'eager'")
        self.cfg, self.glue, self.weights = cfg, glue, weights
        dev = torch.device(device)
        mk = StreamingLinear if weights == "packed" else _DenseLinear
        self.layers = torch.nn.ModuleList()
        max_n = 0
        for li in range(cfg.n_layers):
            pl = packed_layers[li]
            if weights == "packed":
                # linears that share their input are one resident tensor and one launch
                mods = torch.nn.ModuleDict({"qkv": FusedPackedLinear([pl["q_proj"], pl["k_proj"], pl["v_proj"]]),
                                            "o_proj": mk(pl["o_proj"]),
                                            "gate_up": FusedPackedLinear([pl["gate_proj"], pl["up_proj"]]),
                                            "down_proj": mk(pl["down_proj"])})
                max_n = max([max_n, pl["o_proj"]["N"], pl["down_proj"]["N"], mods["qkv"].res.N, mods["gate_up"].res.N])
            else:
                mods = torch.nn.ModuleDict({n: mk(pl[n]) for n in LINEARS})
            self.layers.append(mods)
        if weights == "packed":
            # one shared decode buffer for inputs of more than 8 rows (prefill), like the streaming engine
            self._shared = torch.empty(max_n, dtype=torch.bfloat16, device=dev)
            for mods in self.layers:
                for m in mods.values():
                    m._set_shared_buf(self._shared)
        ones = torch.ones(cfg.hidden, dtype=torch.bfloat16, device=dev)
        self.ln1 = [ones.clone() if norms is None else norms[i][0].to(dev) for i in range(cfg.n_layers)]
        self.ln2 = [ones.clone() if norms is None else norms[i][1].to(dev) for i in range(cfg.n_layers)]
        self.ln_f = ones.clone()
        self.embed = embed.to(dev, torch.bfloat16)
        self.lm_head = lm_head.to(dev, torch.bfloat16)
        half = cfg.head_dim // 2
        inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, half, dtype=torch.float32) / half))
        ang = torch.arange(cfg.max_seq, dtype=torch.float32)[:, None] * inv[None, :]
        self.cos = ang.cos().to(dev)
        self.sin = ang.sin().to(dev)
        self.k_cache = torch.zeros(cfg.n_layers, cfg.max_seq, cfg.n_kv_heads, cfg.head_dim, dtype=torch.bfloat16, device=dev)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.key_pos = torch.arange(cfg.max_seq, device=dev)
        # static inputs / outputs of the captured step
        self.tok = torch.zeros(1, dtype=torch.long, device=dev)
        self.pos = torch.zeros(1, dtype=torch.long, device=dev)
        self.pos32 = torch.zeros(1, dtype=torch.int32, device=dev)
        self.logits = None
        self.graph = None
        if glue == "kernels":
            from .glue import AttnDecode

            bf = dict(dtype=torch.bfloat16, device=dev)
            qd, kd = cfg.n_heads * cfg.head_dim, cfg.n_kv_heads * cfg.head_dim
            # static activations of the one-row step
            self._h = torch.zeros(1, cfg.hidden, **bf)
            self._xn = torch.zeros(1, cfg.hidden, **bf)
            if weights == "packed":                                # outputs of the fused linears and the parts' views
                self._qkv = torch.zeros(1, self.layers[0]["qkv"].res.out_f, **bf)
                self._q, self._k, self._v = self.layers[0]["qkv"].res.split(self._qkv)
                self._gu = torch.zeros(1, self.layers[0]["gate_up"].res.out_f, **bf)
                self._g, self._u = self.layers[0]["gate_up"].res.split(self._gu)
            else:
                self._q, self._k, self._v = torch.zeros(qd, **bf), torch.zeros(kd, **bf), torch.zeros(kd, **bf)
                self._g, self._u = torch.zeros(cfg.intermediate, **bf), torch.zeros(cfg.intermediate, **bf)
            self._a = torch.zeros(1, qd, **bf)
            self._d = torch.zeros(1, cfg.hidden, **bf)             # output of o_proj / down_proj: the next residual
            self._act = torch.zeros(1, cfg.intermediate, **bf)
            self._attn = AttnDecode(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, dev)

    # ------------------------------------------------------------------ core
    def _rope(self, x, pos):
        """x [T, heads, head_dim], pos [T] (rotate-half convention)"""
        c = self.cos.index_select(0, pos)[:, None, :]
        s = self.sin.index_select(0, pos)[:, None, :]
        x1, x2 = x.float().chunk(2, dim=-1)
        return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(x.dtype)

    def _block(self, li, h, pos):
        """h [T, hidden], pos [T] absolute positions (T = 1 in the decode step)"""
        cfg, m = self.cfg, self.layers[li]
        t = h.shape[0]
        x = _rms(h, self.ln1[li], cfg.rms_eps)
        q, k, v = m["qkv"](x) if self.weights == "packed" else (m["q_proj"](x), m["k_proj"](x), m["v_proj"](x))
        q = q.reshape(t, cfg.n_heads, cfg.head_dim)
        k = k.reshape(t, cfg.n_kv_heads, cfg.head_dim)
        v = v.reshape(t, cfg.n_kv_heads, cfg.head_dim)
        q, k = self._rope(q, pos), self._rope(k, pos)
        self.k_cache[li].index_copy_(0, pos, k)
        self.v_cache[li].index_copy_(0, pos, v)
        # attention of the T new queries over the whole static cache, masked to keys <= query position
        rep = cfg.n_heads // cfg.n_kv_heads
        kk = self.k_cache[li].repeat_interleave(rep, dim=1).transpose(0, 1)      # [heads, S, d]
        vv = self.v_cache[li].repeat_interleave(rep, dim=1).transpose(0, 1)
        mask = self.key_pos[None, :] <= pos[:, None]                               # [T, S]
        a = F.scaled_dot_product_attention(q.transpose(0, 1), kk, vv, attn_mask=mask[None])
        a = a.transpose(0, 1).reshape(t, cfg.n_heads * cfg.head_dim)
        h = h + m["o_proj"](a)
        x = _rms(h, self.ln2[li], cfg.rms_eps)
        g, u = m["gate_up"](x) if self.weights == "packed" else (m["gate_proj"](x), m["up_proj"](x))
        return h + m["down_proj"](F.silu(g) * u)

    def _lin(self, li, name, x, out):
        m = self.layers[li][name]
        if self.weights == "packed":
            return m._res.gemv(x, out=out) if m._res is not None else out.copy_(m(x))
        return torch.matmul(x, m.weight.t(), out=out.view(1, -1))

    def _qkv_step(self, li):
        if self.weights == "packed":
            return self.layers[li]["qkv"].res.gemv(self._xn, out=self._qkv)
        for n, o in (("q_proj", self._q), ("k_proj", self._k), ("v_proj", self._v)):
            self._lin(li, n, self._xn, o)

    def _gate_up_step(self, li):
        if self.weights == "packed":
            return self.layers[li]["gate_up"].res.gemv(self._xn, out=self._gu)
        self._lin(li, "gate_proj", self._xn, self._g)
        self._lin(li, "up_proj", self._xn, self._u)

    def _step_kernels(self):
        """One row at position self.pos32 (device) through all layers on the glue kernels; static buffers only."""
        from . import glue as G

        cfg = self.cfg
        torch.index_select(self.embed, 0, self.tok, out=self._h)
        delta = None
        for li in range(cfg.n_layers):
            G.add_rmsnorm(self._h, delta, self.ln1[li], cfg.rms_eps, out=self._xn)
            self._qkv_step(li)
            G.rope_kv(self._q, self._k, self._v, self.pos32, self.k_cache[li], self.v_cache[li], self.cos, self.sin,
                      cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
            self._attn(self._q, self.k_cache[li], self.v_cache[li], self.pos32, out=self._a)
            self._lin(li, "o_proj", self._a, self._d)
            G.add_rmsnorm(self._h, self._d, self.ln2[li], cfg.rms_eps, out=self._xn)
            self._gate_up_step(li)
            G.swiglu(self._g, self._u, out=self._act[0])
            self._lin(li, "down_proj", self._act, self._d)
            delta = self._d
        G.add_rmsnorm(self._h, delta, self.ln_f, cfg.rms_eps, out=self._xn)
        return F.linear(self._xn, self.lm_head).float()

    def _forward(self, tok, pos):
        if self.glue == "kernels" and tok.numel() == 1 and tok.data_ptr() == self.tok.data_ptr():
            return self._step_kernels()
        h = self.embed.index_select(0, tok)
        for li in range(self.cfg.n_layers):
            h = self._block(li, h, pos)
        h = _rms(h[-1:], self.ln_f, self.cfg.rms_eps)
        return F.linear(h, self.lm_head).float()

    # ------------------------------------------------------------------- API
    # Rows of a prompt that go through a layer together on packed weights.  Every pass decodes the layer's weights to bf16
    # once (about 32 us for the four linears of a 1B-class layer, as much as the matmuls of 400 rows), so a pass is as
    # long as its activations allow: 2048 rows of the widest fused linear (gate|up, 34816 columns) are 143 MB.
    PREFILL_ROWS = 2048

    def _prefill_kernels(self, ids, start: int, last: bool):
        """Rows start .. start + T - 1 of a prompt through all layers on the glue kernels; the last row's logits."""
        from . import glue as G

        cfg, t = self.cfg, ids.numel()
        d, qd = cfg.head_dim, cfg.n_heads * cfg.head_dim
        h = self.embed.index_select(0, ids)
        pos0 = torch.full((1,), start, dtype=torch.int32, device=h.device)
        xn = torch.empty_like(h)
        a = torch.empty(t, qd, dtype=torch.bfloat16, device=h.device)
        act = torch.empty(t, cfg.intermediate, dtype=torch.bfloat16, device=h.device)
        delta = None
        for li, m in enumerate(self.layers):
            G.add_rmsnorm(h, delta, self.ln1[li], cfg.rms_eps, out=xn)
            q, k, v = m["qkv"](xn)
            kc, vc = self.k_cache[li], self.v_cache[li]
            G.rope_kv(q, k, v, pos0, kc, vc, self.cos, self.sin, cfg.n_heads, cfg.n_kv_heads, d)
            G.attn_prefill(q, kc, vc, start, cfg.n_heads, cfg.n_kv_heads, d, out=a)
            G.add_rmsnorm(h, m["o_proj"](a), self.ln2[li], cfg.rms_eps, out=xn)
            g, u = m["gate_up"](xn)
            G.swiglu(g, u, out=act)
            delta = m["down_proj"](act)
        if not last:
            return None
        G.add_rmsnorm(h[-1:], delta[-1:], self.ln_f, cfg.rms_eps, out=xn[-1:])
        return F.linear(xn[-1:], self.lm_head).float()

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor, chunk: int | None = None) -> torch.Tensor:
        """Run the prompt through the model (many rows per linear: decode +
        dense matmul path); returns the logits of the last prompt token.
        chunk: the most rows that go through the model together, which bounds the memory of a pass's activations.  None:
        PREFILL_ROWS on the glue kernels, 256 on the eager path (whose score matrices take rows * max_seq)."""
        logits = None
        if self.weights == "packed" and self.glue == "kernels" and self.cfg.head_dim in (64, 128):
            rows, n = self.PREFILL_ROWS if chunk is None else chunk, ids.numel()
            ids = ids.to(self.tok.device)
            for s in range(0, n, rows):
                logits = self._prefill_kernels(ids[s:s + rows], s, s + rows >= n)
            return logits
        chunk = 256 if chunk is None else chunk
        for s in range(0, ids.numel(), chunk):
            part = ids[s:s + chunk].to(self.tok.device)
            pos = torch.arange(s, s + part.numel(), device=part.device)
            logits = self._forward(part, pos)
        return logits

    @torch.no_grad()
    def capture(self):
        """Capture one token step (static tok/pos in, static logits out)."""
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                self._forward(self.tok, self.pos)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self._forward(self.tok, self.pos)
        return self

    @torch.no_grad()
    def step(self, tok: torch.Tensor, pos: int) -> torch.Tensor:
        """One decode step at absolute position `pos`; returns logits [1, vocab]
        (a static tensor when the step is graph-captured)."""
        self.tok.copy_(tok.reshape(1))
        self.pos.fill_(pos)
        self.pos32.fill_(pos)
        if self.graph is not None:
            self.graph.replay()
            return self.logits
        return self._forward(self.tok, self.pos)

    @torch.no_grad()
    def generate(self, prompt_ids: torch.Tensor, n_new: int) -> torch.Tensor:
        """Greedy decode of n_new tokens after the prompt."""
        logits = self.prefill(prompt_ids)
        out = []
        pos = prompt_ids.numel()
        tok = logits.argmax(-1)
        for _ in range(n_new):
            out.append(tok.clone())
            logits = self.step(tok, pos)
            tok = logits.argmax(-1)
            pos += 1
        return torch.cat(out)


class Verifier:
    """T new tokens of ONE sequence in one pass (the verification forward of speculative decoding,
    ixrun/mtp.py:198-280: the draft's tokens go through the model together and the longest prefix that the model's own
    arg-max confirms is kept).  Every packed linear sees T rows (fused GEMV for T <= 8, tensor-core GEMM up to 64), the
    keys and values of the T positions are written into the sequence's cache, and query r attends up to position
    pos0 + r.  Runs on the model's own cache: a rejected tail is simply overwritten by the next call."""

    def __init__(self, model: PackedLlama, rows: int):
        from .glue import AttnDecode

        if model.weights != "packed" or model.glue != "kernels":
            raise ValueError("the verifier runs on packed weights and the glue kernels")
        if not 1 <= rows <= 64:
            raise ValueError("1..64 rows")
        self.m, self.t = model, int(rows)
        cfg, dev = model.cfg, model.embed.device
        bf = dict(dtype=torch.bfloat16, device=dev)
        t = self.t
        first = model.layers[0]
        self._h, self._xn, self._d = (torch.zeros(t, cfg.hidden, **bf) for _ in range(3))
        self._qkv = torch.zeros(t, first["qkv"].res.out_f, **bf)
        self._q, self._k, self._v = (self._qkv[:, a:a + n] for a, n in first["qkv"].res.sections)
        self._gu = torch.zeros(t, first["gate_up"].res.out_f, **bf)
        self._g, self._u = (self._gu[:, a:a + n] for a, n in first["gate_up"].res.sections)
        self._a = torch.zeros(t, cfg.n_heads * cfg.head_dim, **bf)
        self._act = torch.zeros(t, cfg.intermediate, **bf)
        self._attn = AttnDecode(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, dev, splits=model._attn.splits, batch=t)
        self.tok = torch.zeros(t, dtype=torch.long, device=dev)
        self.pos0 = torch.zeros(1, dtype=torch.int32, device=dev)                 # position of the first row
        self.pos_rows = torch.zeros(t, dtype=torch.int32, device=dev)             # pos0 + r
        self._ramp = torch.arange(t, dtype=torch.int32, device=dev)
        self.logits = None
        self.graph = None

    def _lin(self, res, x, out):
        return res.gemv(x, out=out) if self.t <= 8 else res.gemm(x, out=out)

    def _forward(self):
        from . import glue as G

        m, cfg = self.m, self.m.cfg
        torch.add(self._ramp, self.pos0, out=self.pos_rows)
        torch.index_select(m.embed, 0, self.tok, out=self._h)
        delta = None
        for li in range(cfg.n_layers):
            L = m.layers[li]
            G.add_rmsnorm(self._h, delta, m.ln1[li], cfg.rms_eps, out=self._xn)
            self._lin(L["qkv"].res, self._xn, self._qkv)
            G.rope_kv(self._q, self._k, self._v, self.pos0, m.k_cache[li], m.v_cache[li], m.cos, m.sin,
                      cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)              # rows = consecutive positions pos0 + r
            self._attn(self._q, m.k_cache[li], m.v_cache[li], self.pos_rows, out=self._a, q_stride=self._qkv.shape[1],
                       shared_cache=True)
            self._lin(L["o_proj"]._res, self._a, self._d)
            G.add_rmsnorm(self._h, self._d, m.ln2[li], cfg.rms_eps, out=self._xn)
            self._lin(L["gate_up"].res, self._xn, self._gu)
            G.swiglu(self._g, self._u, out=self._act)
            self._lin(L["down_proj"]._res, self._act, self._d)
            delta = self._d
        G.add_rmsnorm(self._h, delta, m.ln_f, cfg.rms_eps, out=self._xn)
        return F.linear(self._xn, m.lm_head).float()

    @torch.no_grad()
    def capture(self):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                self._forward()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self._forward()
        return self

    @torch.no_grad()
    def __call__(self, tokens: torch.Tensor, pos0: int) -> torch.Tensor:
        """tokens [T] at positions pos0 .. pos0 + T - 1; returns logits [T, vocab] (row r = the model's prediction for
        position pos0 + r + 1)."""
        self.tok.copy_(tokens.reshape(self.t))
        self.pos0.fill_(pos0)
        if self.graph is not None:
            self.graph.replay()
            return self.logits
        return self._forward()

    @torch.no_grad()
    def accept(self, tokens: torch.Tensor, pos0: int):
        """tokens[0] is the last confirmed token, tokens[1:] a draft of what follows.  Returns (number of draft tokens the
        model's greedy arg-max confirms, the model's own next token after the confirmed prefix)."""
        pred = self(tokens, pos0).argmax(-1)                          # pred[r]: greedy token for position pos0 + r + 1
        ok = (pred[:-1] == tokens[1:].to(pred.device)).long().cumprod(0)
        n = int(ok.sum().item())
        return n, pred[n]


class BatchedGreedyDecoder:
    """B sequences decoded in lock-step on a packed model: the decode loop of the reference's batched generator
    (ixrun/batching.py:88-234: per-row greedy arg-max, sequences of different lengths, one KV cache per row) without its
    request queue and tokenizer.  Every packed linear sees B rows per step -- the fused GEMV for B <= 8, the tensor-core
    GEMM on the resident layout up to 64 -- and the glue kernels take one row per sequence (its own position, its own
    cache).  One step is one CUDA graph."""

    def __init__(self, model: PackedLlama, batch: int):
        from .glue import AttnDecode

        if model.weights != "packed" or model.glue != "kernels":
            raise ValueError("the batched decoder runs on packed weights and the glue kernels")
        if not 1 <= batch <= 64:
            raise ValueError("1..64 sequences")
        self.m, self.b = model, int(batch)
        cfg, dev = model.cfg, model.embed.device
        bf = dict(dtype=torch.bfloat16, device=dev)
        b = self.b
        self.k_cache = torch.zeros(cfg.n_layers, b, cfg.max_seq, cfg.n_kv_heads, cfg.head_dim, **bf)
        self.v_cache = torch.zeros_like(self.k_cache)
        qd = cfg.n_heads * cfg.head_dim
        first = model.layers[0]
        self._h, self._xn, self._d = (torch.zeros(b, cfg.hidden, **bf) for _ in range(3))
        self._qkv = torch.zeros(b, first["qkv"].res.out_f, **bf)
        self._q, self._k, self._v = (self._qkv[:, a:a + n] for a, n in first["qkv"].res.sections)
        self._gu = torch.zeros(b, first["gate_up"].res.out_f, **bf)
        self._g, self._u = (self._gu[:, a:a + n] for a, n in first["gate_up"].res.sections)
        self._a = torch.zeros(b, qd, **bf)
        self._act = torch.zeros(b, cfg.intermediate, **bf)
        # the same context splits as the one-sequence step: a sequence then gets the same bits alone or in a batch
        self._attn = AttnDecode(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, dev, splits=model._attn.splits, batch=b)
        self.tok = torch.zeros(b, dtype=torch.long, device=dev)
        self.pos32 = torch.zeros(b, dtype=torch.int32, device=dev)
        self.logits = None
        self.graph = None

    def _lin(self, res, x, out):
        return res.gemv(x, out=out) if self.b <= 8 else res.gemm(x, out=out)

    def _step_kernels(self):
        from . import glue as G

        m, cfg = self.m, self.m.cfg
        torch.index_select(m.embed, 0, self.tok, out=self._h)
        delta = None
        for li in range(cfg.n_layers):
            L = m.layers[li]
            G.add_rmsnorm(self._h, delta, m.ln1[li], cfg.rms_eps, out=self._xn)
            self._lin(L["qkv"].res, self._xn, self._qkv)
            G.rope_kv(self._q, self._k, self._v, self.pos32, self.k_cache[li], self.v_cache[li], m.cos, m.sin,
                      cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, batched=True)
            self._attn(self._q, self.k_cache[li], self.v_cache[li], self.pos32, out=self._a, q_stride=self._qkv.shape[1])
            self._lin(L["o_proj"]._res, self._a, self._d)
            G.add_rmsnorm(self._h, self._d, m.ln2[li], cfg.rms_eps, out=self._xn)
            self._lin(L["gate_up"].res, self._xn, self._gu)
            G.swiglu(self._g, self._u, out=self._act)
            self._lin(L["down_proj"]._res, self._act, self._d)
            delta = self._d
        G.add_rmsnorm(self._h, delta, m.ln_f, cfg.rms_eps, out=self._xn)
        return F.linear(self._xn, m.lm_head).float()

    @torch.no_grad()
    def prefill(self, prompts: list) -> torch.Tensor:
        """Run every prompt through the model (the many-row path), keep its keys and values in the row's own cache;
        returns the first generated token of every sequence [B]."""
        if len(prompts) != self.b:
            raise ValueError(f"{self.b} prompts expected")
        first = []
        for r, ids in enumerate(prompts):
            logits = self.m.prefill(ids)
            n = ids.numel()
            self.k_cache[:, r, :n] = self.m.k_cache[:, :n]
            self.v_cache[:, r, :n] = self.m.v_cache[:, :n]
            self.pos32[r] = n
            first.append(logits.argmax(-1))
        return torch.cat(first)

    @torch.no_grad()
    def capture(self):
        saved = self.pos32.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                self._step_kernels()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self._step_kernels()
        self.pos32.copy_(saved)
        return self

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Feed one token per sequence (at the sequences' current positions); returns logits [B, vocab]."""
        self.tok.copy_(tokens.reshape(self.b))
        if self.graph is not None:
            self.graph.replay()
            out = self.logits
        else:
            out = self._step_kernels()
        self.pos32 += 1
        return out

    @torch.no_grad()
    def generate(self, prompts: list, n_new: int) -> torch.Tensor:
        """Greedy decode of n_new tokens for every prompt; returns [B, n_new]."""
        tok = self.prefill(prompts)
        out = []
        for _ in range(n_new):
            out.append(tok.clone())
            tok = self.step(tok).argmax(-1)
        return torch.stack(out, dim=1)


class PagedDecoder:
    """Requests that come and go, decoded together on a packed model over a paged KV cache: what the reference's batched
    generator does with one static cache row per sequence (ixrun/batching.py:88-234), for requests of different lengths in
    memory for the tokens that there are.  A step feeds every request the tokens that it has and the model has not seen: the
    next piece of its prompt, or its last token.  Steps of single tokens are one CUDA graph (``capture``).  Per request:
    penalties, biases and a mask of allowed tokens; the token is the arg-max behind them.  Steps of several decoders of one model,
    which share its buffer for decoded weights, must not overlap."""

    def __init__(self, model: PackedLlama, requests: int, n_pages: int, page: int = 64, max_bias: int = 64):
        from .logits import MAX_BIASES, MAX_TOKENS, MAX_VOCAB
        from .paged import AttnPaged, PageTables

        if model.weights != "packed" or model.glue != "kernels":
            raise ValueError("the paged decoder runs on packed weights and the glue kernels")
        if not 1 <= requests <= 64:
            raise ValueError("1..64 requests")
        if not 0 <= max_bias <= MAX_BIASES:
            raise ValueError(f"0..{MAX_BIASES} biases")
        if model.cfg.vocab > MAX_VOCAB or model.cfg.max_seq >= MAX_TOKENS:
            raise ValueError(f"a vocabulary of at most {MAX_VOCAB}, less than {MAX_TOKENS} tokens of a request")
        self.m, self.b = model, int(requests)
        cfg, dev, b = model.cfg, model.embed.device, self.b
        self._attn = AttnPaged(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, dev)
        self.pages = PageTables(b, n_pages, page, -(-cfg.max_seq // page), dev)
        self.k_pages = torch.zeros(cfg.n_layers, n_pages, page, cfg.n_kv_heads, cfg.head_dim, dtype=torch.bfloat16, device=dev)
        self.v_pages = torch.zeros_like(self.k_pages)
        # what is known of every request: its tokens (prompt and answer), how many, and its rules
        ints = dict(dtype=torch.int32, device=dev)
        self.history = torch.zeros(b, cfg.max_seq + 1, **ints)
        self.n_tokens, self.n_prompt, self.q_len = (torch.zeros(b, **ints) for _ in range(3))
        self.repetition, self.presence, self.frequency = (torch.zeros(b, dtype=torch.float32, device=dev) for _ in range(3))
        self.repetition.fill_(1.0)
        self.bias_ids = torch.full((b, max_bias), -1, **ints)
        self.bias_values = torch.zeros(b, max_bias, dtype=torch.float32, device=dev)
        self.mask = torch.zeros(b, -(-cfg.vocab // 32), **ints)
        self.mask_row = torch.full((b,), -1, **ints)
        # results of a step: logits behind the rules, and the token of every request (-1: none in this step)
        self.logits = torch.zeros(b, cfg.vocab, dtype=torch.float32, device=dev)
        self.token = torch.full((b,), -1, dtype=torch.long, device=dev)
        self._best = torch.zeros(b, dtype=torch.long, device=dev)
        # the host's account of the same: tokens known (None: no request), tokens in the cache, tokens that a bias bans; pages left
        self._known, self._cached, self._banned = [None] * b, [0] * b, [[]] * b
        self._pages_left, self._fed = n_pages, [0] * b
        # steps made, the one in which a request last had rows (or was added), and the requests' order
        self._steps, self._last, self._came, self._added = 0, [0] * b, [0] * b, 0
        self._step, self._bufs = self.pages.new_step(b), self._buffers(b)
        self.graph = None

    def _buffers(self, rows):
        cfg, first = self.m.cfg, self.m.layers[0]
        new = lambda n: torch.zeros(rows, n, dtype=torch.bfloat16, device=self.m.embed.device)  # noqa: E731
        return dict(h=new(cfg.hidden), xn=new(cfg.hidden), d=new(cfg.hidden), qkv=new(first["qkv"].res.out_f), gu=new(first["gate_up"].res.out_f),
                    a=new(cfg.n_heads * cfg.head_dim), act=new(cfg.intermediate))

    def _lin(self, res, x, out):
        if x.shape[0] <= 8:
            return res.gemv(x, out=out)
        if x.shape[0] <= 64:
            return res.gemm(x, out=out)
        return torch.matmul(x, res.decode(out=self.m._shared[:res.N], kind="bf16").t(), out=out)

    def _forward(self, step, bufs, max_q):
        """One pass of the rows that `step` says through the model; logits, tokens and what is known of the requests."""
        from . import glue as G
        from .logits import apply_rules
        from .paged import rope_kv_paged

        m, cfg = self.m, self.m.cfg
        self.pages.step(self.q_len, step.slot.numel(), out=step)
        h, xn, d, a, act = (bufs[n] for n in ("h", "xn", "d", "a", "act"))
        q, k, v = (bufs["qkv"][:, o:o + n] for o, n in m.layers[0]["qkv"].res.sections)
        g, u = (bufs["gu"][:, o:o + n] for o, n in m.layers[0]["gate_up"].res.sections)
        at = step.owner.clamp(min=0).long() * self.history.shape[1] + step.pos     # (rows behind the last token: any token)
        torch.index_select(m.embed, 0, self.history.view(-1).index_select(0, at).long(), out=h)
        delta = None
        for li, L in enumerate(m.layers):
            G.add_rmsnorm(h, delta, m.ln1[li], cfg.rms_eps, out=xn)
            self._lin(L["qkv"].res, xn, bufs["qkv"])
            rope_kv_paged(q, k, v, step.pos, step.slot, self.k_pages[li], self.v_pages[li], m.cos, m.sin, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
            self._attn(q, self.k_pages[li], self.v_pages[li], self.pages.table, step.length, step.cu_rows, max_q=max_q, out=a)
            self._lin(L["o_proj"]._res, a, d)
            G.add_rmsnorm(h, d, m.ln2[li], cfg.rms_eps, out=xn)
            self._lin(L["gate_up"].res, xn, bufs["gu"])
            G.swiglu(g, u, out=act)
            self._lin(L["down_proj"]._res, act, d)
            delta = d
        last = (step.cu_rows[1:] - 1).clamp(min=0)                                 # (requests without a row: any row)
        x = G.add_rmsnorm(h.index_select(0, last), delta.index_select(0, last), m.ln_f, cfg.rms_eps)
        apply_rules(F.linear(x, m.lm_head), self.history, self.n_tokens, self.n_prompt, self.repetition, self.presence, self.frequency,
                    self.bias_ids if self.bias_ids.shape[1] else None, self.bias_values if self.bias_ids.shape[1] else None, self.mask,
                    self.mask_row, out=self.logits, token=self._best)
        # a request whose known tokens are all in the cache has a new one
        new = (self.q_len > 0) & (step.length == self.n_tokens)
        end = self.n_tokens.long().clamp(max=self.history.shape[1] - 1)[:, None]   # (of a full request: rewritten as it is)
        self.history.scatter_(1, end, torch.where(new[:, None], self._best[:, None].int(), self.history.gather(1, end)))
        self.n_tokens += new
        self.token.copy_(torch.where(new, self._best, -1))

    # ------------------------------------------------------------------- API
    def _request(self, r):
        if not 0 <= r < self.b or self._known[r] is None:
            raise ValueError(f"no request {r}")
        return r

    def _checked(self, prompt, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
        """the checks of ``add``; returns the biases' values and the tokens that they ban"""
        if not 1 <= prompt.numel() <= self.m.cfg.max_seq:
            raise ValueError(f"a prompt of 1..{self.m.cfg.max_seq} tokens")
        if prompt.is_floating_point() or prompt.min() < 0 or prompt.max() >= self.m.cfg.vocab:
            raise ValueError(f"tokens are whole numbers of 0..{self.m.cfg.vocab - 1}")
        penalties = torch.tensor([repetition, presence, frequency], dtype=torch.float32)
        if not penalties[0] > 0.0 or not penalties.isfinite().all():
            raise ValueError("repetition must be positive, penalties finite")
        bias = bias or {}
        if len(bias) > self.bias_ids.shape[1]:
            raise ValueError(f"at most {self.bias_ids.shape[1]} biases")
        values = torch.tensor(list(bias.values()), dtype=torch.float32)
        if values.isnan().any():
            raise ValueError("a bias is a number")
        banned = [t for t, x in zip(bias, values.tolist()) if x == -math.inf and 0 <= t < self.m.cfg.vocab]
        self._check_allowed(allowed, banned)
        return values, banned

    @torch.no_grad()
    def add(self, prompt: torch.Tensor, repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0, bias: dict | None = None,
            allowed: torch.Tensor | None = None) -> int:
        """Takes a request in; returns its number (a free one).  The rules are those of ``logits.apply_rules``, penalties finite; bias:
        {token: value}; allowed: a bool tensor [vocab].  Rules that leave no token (none allowed that has no bias of -inf) are
        refused."""
        if None not in self._known:
            raise RuntimeError("all requests are taken")
        values, banned = self._checked(prompt, repetition, presence, frequency, bias, allowed)
        n, r = prompt.numel(), self._known.index(None)
        self._banned[r] = banned
        self._allow(r, allowed)
        dev = self.history.device
        self.history[r, :n].copy_(prompt.reshape(-1))
        for t, x in ((self.n_tokens, n), (self.n_prompt, n), (self.repetition, repetition), (self.presence, presence), (self.frequency, frequency)):
            t[r].fill_(x)
        if self.bias_ids.shape[1]:
            self.bias_ids[r].fill_(-1)
        if bias:
            self.bias_ids[r, :len(bias)].copy_(torch.tensor(list(bias), dtype=torch.int32, device=dev))
            self.bias_values[r, :len(bias)].copy_(values)
        self._known[r], self._cached[r], self._last[r], self._came[r] = n, 0, self._steps, self._added
        self._added += 1
        return r

    def allow(self, r: int, allowed: torch.Tensor | None):
        """The tokens that request r may have from now on (a bool tensor [vocab]; None: all), as a grammar moves on.  At least one."""
        self._check_allowed(allowed, self._banned[self._request(r)])
        self._allow(r, allowed)

    def _check_allowed(self, allowed, banned):
        """refuses what leaves no token (the arg-max of a row of -inf would be token 0); banned: tokens with a bias of -inf"""
        vocab = self.m.cfg.vocab
        if allowed is not None and (allowed.dtype != torch.bool or allowed.shape != (vocab,)):
            raise ValueError("allowed: a bool tensor [vocab]")
        left = vocab - len(banned) if allowed is None else int(allowed.sum()) - (int(allowed[banned].sum()) if banned else 0)
        if left < 1:
            raise ValueError("the rules leave no token")

    @torch.no_grad()
    def _allow(self, r, allowed):
        if allowed is None:
            self.mask_row[r].fill_(-1)
            return
        bits = F.pad(allowed.to(self.mask.device), (0, self.mask.shape[1] * 32 - allowed.numel())).view(-1, 32).long()
        words = (bits << torch.arange(32, device=bits.device)).sum(1)
        self.mask[r].copy_(torch.where(words >= 2**31, words - 2**32, words))
        self.mask_row[r].fill_(r)

    @torch.no_grad()
    def remove(self, r: int):
        """The request's pages go back to the pool, and its number may be taken by the next one."""
        self._request(r)
        done = torch.zeros(self.b, dtype=torch.bool, device=self.history.device)
        done[r].fill_(True)
        self.pages.release(done)
        self.n_tokens[r].fill_(0)
        self._pages_left += self._n_pages(self._cached[r])
        self._known[r], self._cached[r] = None, 0

    def _n_pages(self, tokens):
        return -(-tokens // self.pages.page)

    def _share(self, max_rows):
        """rows of every request in a step of at most max_rows"""
        left, q_len = int(max_rows), [0] * self.b
        todo = {r: n - self._cached[r] for r, n in enumerate(self._known) if n is not None}
        singles = sorted((r for r in todo if todo[r] == 1), key=lambda r: (self._last[r], r))
        prompts = sorted((r for r in todo if todo[r] > 1), key=lambda r: self._came[r])
        waited = [r for r in prompts[:1] if self._last[r] < self._steps]
        for r in waited + singles + prompts[len(waited):]:
            q_len[r] = min(todo[r], left)
            left -= q_len[r]
        return q_len

    def _account(self, q_len):
        """what a step of these rows has done"""
        self._steps += 1
        for r, n in enumerate(q_len):
            if not n:
                continue
            self._last[r] = self._steps
            self._cached[r] += n
            if self._cached[r] == self._known[r]:
                self._known[r] += 1

    @torch.no_grad()
    def step(self, max_rows: int = PackedLlama.PREFILL_ROWS) -> torch.Tensor:
        """Feeds the requests what they have, at most max_rows rows in all: single tokens first, those that have waited longest before
        others, then prompts in the order in which they were added; the first of these comes before the single tokens where it had
        no row in the step before.  So every request gets on, however few rows there are.  Returns tokens int64 [requests], -1
        for those without a new one (a static tensor).  RuntimeError, and nothing launched, where there is nothing to feed, a
        request has all max_seq tokens, or the pages do not suffice."""
        if max_rows < 1:
            raise ValueError("max_rows must be positive")
        q_len = self._share(max_rows)
        if not any(q_len):
            raise RuntimeError("no request to feed")
        if any(self._cached[r] + n > self.m.cfg.max_seq for r, n in enumerate(q_len)):
            raise RuntimeError(f"a request has all {self.m.cfg.max_seq} tokens that fit: remove it")
        need = sum(self._n_pages(c + n) - self._n_pages(c) for c, n in zip(self._cached, q_len))
        if need > self._pages_left:
            raise RuntimeError(f"the step needs {need} pages, {self._pages_left} are left: remove a request")
        if q_len != self._fed:
            self.q_len.copy_(torch.tensor(q_len, dtype=torch.int32))
            self._fed = q_len
        if max(q_len) == 1:
            if self.graph is not None:
                self.graph.replay()
            else:
                self._forward(self._step, self._bufs, 1)
        else:
            self._forward(self.pages.new_step(sum(q_len)), self._buffers(sum(q_len)), max(q_len))
        self._pages_left -= need
        self._account(q_len)
        return self.token

    @torch.no_grad()
    def capture(self):
        """Captures the step of single tokens."""
        self.q_len.zero_()                     # (the warm-up feeds nothing)
        self._fed = [0] * self.b
        with torch.cuda.device(self.q_len.device):         # (a capture takes what runs on the current device)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(2):
                    self._forward(self._step, self._bufs, 1)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self._forward(self._step, self._bufs, 1)
        return self

    @torch.no_grad()
    def generate(self, prompts: list, n_new: int, eos: int | None = None, max_rows: int = PackedLlama.PREFILL_ROWS, **rules) -> list:
        """n_new tokens for every prompt (fewer for one that ends with eos or has all max_seq tokens), as lists; a prompt waits
        until a number and the pages for its whole answer are free."""
        if n_new < 1 or max_rows < 1:
            raise ValueError("n_new and max_rows must be positive")
        if any(n is not None for n in self._known):
            raise RuntimeError("generate wants the decoder for itself: remove the requests that are there")
        for ids in prompts:                            # (before the first one is taken in: a refusal leaves no request behind)
            self._checked(ids, **rules)
        whole = [self._n_pages(min(ids.numel() + n_new - 1, self.m.cfg.max_seq)) for ids in prompts]
        if whole and max(whole) > self._pages_left:
            raise RuntimeError(f"a prompt and its answer need {max(whole)} pages, there are {self._pages_left}")
        out, waiting, running, free = [[] for _ in prompts], list(range(len(prompts))), {}, self._pages_left
        while waiting or running:
            while waiting and None in self._known and whole[waiting[0]] <= free:
                i = waiting.pop(0)
                running[self.add(prompts[i], **rules)] = i
                free -= whole[i]
            tokens = self.step(max_rows).tolist()
            for r, i in list(running.items()):
                if tokens[r] < 0:
                    continue
                out[i].append(tokens[r])
                if len(out[i]) == n_new or tokens[r] == eos or self._known[r] > self.m.cfg.max_seq:
                    self.remove(r)
                    del running[r]
                    free += whole[i]
        return out


def synthetic_llama(cfg: LlamaConfig, seed: int = 0, distinct_layers: bool = True):
    """Random-init weights of the config: Laplace codes for every linear (one
    tensor per linear type and layer when distinct_layers, else one per type
    shared by all layers), N(0, 0.02) embeddings and head."""
    from .synth import synthetic_packed

    shapes = linear_shapes(cfg)
    layers = []
    cache = {}
    for li in range(cfg.n_layers):
        d = {}
        for j, n in enumerate(LINEARS):
            key = (li if distinct_layers else 0, n)
            if key not in cache:
                cache[key] = synthetic_packed(*shapes[n], seed=seed * 1000003 + key[0] * 16 + j)
            d[n] = cache[key]
        layers.append(d)
    g = torch.Generator().manual_seed(seed + 17)
    embed = (torch.randn(cfg.vocab, cfg.hidden, generator=g) * 0.02).bfloat16()
    head = (torch.randn(cfg.vocab, cfg.hidden, generator=g) * 0.02).bfloat16()
    return layers, embed, head
