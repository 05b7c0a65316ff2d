"""Random-init Llama-style text decoder of the SmolLM2-360M shape.

The reference runs the pretrained SmolVLM2 text model (HF LlamaModel) and routes
its attention through GPUCache (src/gpu_cache.py:151-183); the checkpoint is not
part of this build, so this module restates the decoder itself with random
weights: 32 layers, hidden 960, 15 query / 5 KV heads of dim 64, SiLU MLP of
width 2560, RMSNorm eps 1e-5, rotary embeddings (theta 100000), tied embeddings,
bf16. Projections use the joined QKV and gate/up weights of the reference's fused
mode (src/gpu_ops.py:26-47). With a GPUCache the attention is the packed-KV path
(append + attend on the sm_100a kernels); with a NativeCache it is plain bf16
history + SDPA (the reference's "native" mode).

projections='fp8' (CUDA; not in the reference) runs the projections in 8 bits: the
joined weights are e4m3 blocks (half the bytes a step has to stream), the norms write
the e4m3 rows the projections read, and gate, up, SiLU and their product are one
launch. Residual stream, attention, norms' sums, embeddings and logits stay as they are.
Its load_state_dict takes a bf16 decoder's state too and quantises the projections.
"""
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import gpu_kernels as K
from .gpu_cache import GPUCache, RequestBatch, append_many, attend_many
from .gpu_ops import (Fp8, activation_product, add_rms, add_rms_fp8, cuda_rms, fp8_gate_up, fp8_linear, fp8_quantize,
                      fp8_quantize_weight)

PROJECTIONS = ('bf16', 'fp8')


@dataclass(frozen=True)
class DecoderConfig:
    layers: int = 32
    hidden: int = 960
    q_heads: int = 15
    kv_heads: int = 5
    head_dim: int = 64
    intermediate: int = 2560
    vocab: int = 49280
    rms_eps: float = 1e-5
    rope_theta: float = 100000.0
    init_std: float = 0.02


SMOLLM2_360M = DecoderConfig()


class NativeCache:
    """Unquantised bf16 history per layer (the reference's native DynamicCache mode)."""

    def __init__(self, layers):
        self.k = [None] * layers
        self.v = [None] * layers

    def get_seq_length(self, layer_idx=0):
        return 0 if self.k[layer_idx] is None else self.k[layer_idx].shape[2]

    def update(self, k, v, layer):
        self.k[layer] = k if self.k[layer] is None else torch.cat((self.k[layer], k), 2)
        self.v[layer] = v if self.v[layer] is None else torch.cat((self.v[layer], v), 2)
        return self.k[layer], self.v[layer]

    def fork(self):
        other = NativeCache(len(self.k))
        other.k, other.v = list(self.k), list(self.v)  # torch.cat never mutates: sharing is safe
        return other


def rope_tables(cfg, positions, device):
    inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, cfg.head_dim, 2, device=device, dtype=torch.float32) / cfg.head_dim))
    freqs = positions.float()[:, None] * inv[None, :]
    emb = torch.cat((freqs, freqs), dim=-1)
    return emb.cos(), emb.sin()


def apply_rope(x, cos, sin):
    """HF Llama rotate-half rotary embedding over the last dimension (computed in
    fp32; cos / sin broadcast against x)."""
    half = x.shape[-1] // 2
    xf = x.float()
    rot = torch.cat((-xf[..., half:], xf[..., :half]), dim=-1)
    return (xf * cos + rot * sin).to(x.dtype)


class Fp8Weight(torch.nn.Module):
    """8-bit blocks of one bf16 weight [n, k], as buffers."""

    def __init__(self, w):
        super().__init__()
        q, scale = fp8_quantize_weight(w)
        self.register_buffer('q', q)
        self.register_buffer('scale', scale)

    def _apply(self, fn, recurse=True):
        """Moves with its module; casts (to(torch.bfloat16), float()) are for the other weights."""
        q, scale = self.q, self.scale
        super()._apply(fn, recurse)
        if (self.q.dtype, self.scale.dtype) != (q.dtype, scale.dtype):
            self.q, self.scale = q.to(self.q.device), scale.to(self.scale.device)
        return self

    @property
    def blocks(self):
        return Fp8(self.q, self.scale)


class Decoder(torch.nn.Module):
    def __init__(self, cfg=SMOLLM2_360M, device='cuda', dtype=torch.bfloat16, seed=0, projections='bf16'):
        super().__init__()
        if projections not in PROJECTIONS:
            raise ValueError(f'projections must be one of {PROJECTIONS}')
        if projections == 'fp8' and (torch.device(device).type != 'cuda' or dtype != torch.bfloat16):
            raise ValueError('8-bit projections need CUDA and a bfloat16 decoder')
        self.cfg = cfg
        self.fp8 = projections == 'fp8'
        gen = torch.Generator(device='cpu').manual_seed(seed)

        def w(*shape):
            return torch.nn.Parameter((torch.randn(*shape, generator=gen) * cfg.init_std).to(dtype).to(device),
                                      requires_grad=False)

        def per_layer(*shape):  # the same random weights whatever they are held in
            weights = (w(*shape) for _ in range(cfg.layers))
            if self.fp8:
                return torch.nn.ModuleList([Fp8Weight(x) for x in weights])
            return torch.nn.ParameterList(list(weights))

        qkv_out = (cfg.q_heads + 2 * cfg.kv_heads) * cfg.head_dim
        self.embed = w(cfg.vocab, cfg.hidden)
        self.qkv = per_layer(qkv_out, cfg.hidden)
        self.o = per_layer(cfg.hidden, cfg.q_heads * cfg.head_dim)
        if self.fp8:  # gate and up apart: each one's blocks begin at its own first row
            self.register_load_state_dict_pre_hook(Decoder._quantise_state)
            self.gate, self.up = torch.nn.ModuleList(), torch.nn.ModuleList()
            for _ in range(cfg.layers):
                gate, up = w(2 * cfg.intermediate, cfg.hidden).chunk(2)
                self.gate.append(Fp8Weight(gate))
                self.up.append(Fp8Weight(up))
        else:
            self.gate_up = per_layer(2 * cfg.intermediate, cfg.hidden)
        self.down = per_layer(cfg.hidden, cfg.intermediate)
        ones = lambda: torch.nn.Parameter(torch.ones(cfg.hidden, dtype=dtype, device=device), requires_grad=False)
        self.norm_attn = torch.nn.ParameterList([ones() for _ in range(cfg.layers)])
        self.norm_mlp = torch.nn.ParameterList([ones() for _ in range(cfg.layers)])
        self.norm_out = ones()

    def _quantise_state(self, state, prefix, *_):
        """Projections in `state` that a bf16 decoder of this shape holds, as this one's 8-bit blocks."""
        for name, parts in (('qkv', ('qkv',)), ('o', ('o',)), ('gate_up', ('gate', 'up')), ('down', ('down',))):
            for layer in range(self.cfg.layers):
                held = [getattr(self, part)[layer].q for part in parts]
                w = state.get(f'{prefix}{name}.{layer}')
                if w is None:
                    continue
                if w.shape != (sum(q.shape[0] for q in held), held[0].shape[1]):  # loading says which do not fit
                    continue
                del state[f'{prefix}{name}.{layer}']
                for part, q, rows in zip(parts, held, w.detach().split([q.shape[0] for q in held])):
                    blocks = fp8_quantize_weight(rows.to(q.device, torch.bfloat16))
                    state[f'{prefix}{part}.{layer}.q'], state[f'{prefix}{part}.{layer}.scale'] = blocks

    def rms(self, x, weight):
        return cuda_rms(x, weight, self.cfg.rms_eps)

    def add_norm(self, x, y, weight):
        """(x + y, its RMSNorm * weight): the residual add and the next norm of a
        layer in one call (one launch on CUDA); y None: (x, norm of x). With 8-bit
        projections the norm is Fp8 rows."""
        return (add_rms_fp8 if self.fp8 else add_rms)(x, y, weight, self.cfg.rms_eps)

    def mlp(self, h, layer):
        """The gated MLP of one layer's normed input h."""
        if self.fp8:
            return fp8_linear(fp8_gate_up(h, self.gate[layer].blocks, self.up[layer].blocks), self.down[layer].blocks)
        gate, up = F.linear(h, self.gate_up[layer]).chunk(2, dim=-1)
        return F.linear(activation_product(gate, up), self.down[layer])

    def output(self, out, layer):
        """The output projection of one layer's attention out [..., q_heads * head_dim]."""
        if self.fp8:
            return fp8_linear(fp8_quantize(out), self.o[layer].blocks)
        return F.linear(out, self.o[layer])

    def run_layers(self, x, attend):
        """The decoder layers over x: attend(h, layer) is a layer's attention of the
        normed input h, o_proj included. Returns the last residual stream."""
        c = self.cfg
        x, h = self.add_norm(x, None, self.norm_attn[0])
        for layer in range(c.layers):
            x, h = self.add_norm(x, attend(h, layer), self.norm_mlp[layer])
            m = self.mlp(h, layer)
            if layer + 1 < c.layers:
                x, h = self.add_norm(x, m, self.norm_attn[layer + 1])
            else:
                x = x + m
        return x

    def project_qkv(self, x, layer, cos, sin):
        """q [B, q_heads, n, d] and k / v [B, kv_heads, n, d] of x [B, n, hidden] (bf16,
        or Fp8 rows with 8-bit projections): one joined projection and one rotary pass over the query and key heads together
        (cos / sin [B or 1, n, 1, d]); q, k and v are strided views, which the cache
        kernels take as they are."""
        c = self.cfg
        h = fp8_linear(x, self.qkv[layer].blocks) if self.fp8 else F.linear(x, self.qkv[layer])
        b, n = h.shape[0], h.shape[1]
        h = h.view(b, n, c.q_heads + 2 * c.kv_heads, c.head_dim)
        if h.is_cuda:  # one launch, bit-identical to apply_rope
            qk = K.rotary(h, cos, sin, c.q_heads + c.kv_heads)
        else:  # the native-cache decoder on the CPU
            qk = apply_rope(h[:, :, :c.q_heads + c.kv_heads], cos, sin)
        q = qk[:, :, :c.q_heads].transpose(1, 2)
        k = qk[:, :, c.q_heads:].transpose(1, 2)
        v = h[:, :, c.q_heads + c.kv_heads:].transpose(1, 2)
        return q, k, v

    def rotary(self, positions, b, n, device):
        """cos / sin [b, n, 1, d] of positions [b * n] (or [n] for b = 1)."""
        cos, sin = rope_tables(self.cfg, positions.reshape(-1), device)
        return cos.view(b, n, 1, -1), sin.view(b, n, 1, -1)

    def attention(self, x, layer, cache, cos, sin):
        q, k, v = self.project_qkv(x, layer, cos, sin)
        n = q.shape[2]
        if isinstance(cache, GPUCache):
            out = cache.append_attend(q, k, v, layer)  # append + attend in one call; [1, n, q_heads, d]
        else:
            past = cache.get_seq_length(layer)
            kk, vv = cache.update(k, v, layer)
            mask = torch.arange(past + n, device=q.device)[None, :] <= past + torch.arange(n, device=q.device)[:, None]
            out = F.scaled_dot_product_attention(q, kk, vv, attn_mask=mask, enable_gqa=True).transpose(1, 2)
        return self.output(out.reshape(1, n, -1), layer)

    def attention_chunks(self, x, layer, cache, cos, sin):
        """Attention of B token chunks x [B, n, hidden] side by side over the cache's
        history: each chunk sees the history and its own earlier tokens; nothing is
        appended (the packed path runs one batched kernel call per layer)."""
        q, k, v = self.project_qkv(x, layer, cos, sin)
        b, n = q.shape[0], q.shape[2]
        past = cache.get_seq_length(layer)
        if isinstance(cache, GPUCache):
            out = cache.attend_batched(q, k, v, layer, past)  # [B, n, q_heads, d]
        else:
            if past:
                k = torch.cat((cache.k[layer].expand(b, -1, -1, -1), k), 2)
                v = torch.cat((cache.v[layer].expand(b, -1, -1, -1), v), 2)
            mask = torch.arange(past + n, device=q.device)[None, :] <= past + torch.arange(n, device=q.device)[:, None]
            out = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, enable_gqa=True).transpose(1, 2)
        return self.output(out.reshape(b, n, -1), layer)

    def attention_many(self, x, layer, caches, cos, sin):
        """Attention of B requests' frames x [B, n, hidden], request r over caches[r],
        appending each frame's K/V to its own cache (one pack and one attention
        launch for all of them)."""
        q, k, v = self.project_qkv(x, layer, cos, sin)
        b, n = q.shape[0], q.shape[2]
        pasts = append_many(caches, k, v, layer)
        out = attend_many(caches, q, k, v, layer, pasts)  # [B, n, q_heads, d]
        return self.output(out.reshape(b, n, -1), layer)

    def forward_many(self, caches, ids=None, embeds=None, logits=0):
        """forward() for B independent requests stepped together (request batching,
        not in the reference): ids [B, n] or embeds [B, n, hidden], request r appended
        to caches[r] (GPUCache objects with their own pools; their histories may
        differ in length). Returns fp32 logits [B, logits, vocab] (or None)."""
        x = self.embed[ids] if embeds is None else embeds
        b, n = x.shape[0], x.shape[1]
        if len(caches) != b:
            raise ValueError('one cache per request')
        pasts = torch.tensor([c.get_seq_length(0) for c in caches], device=x.device)
        positions = pasts[:, None] + torch.arange(n, device=x.device)[None, :]  # [B, n]
        cos, sin = self.rotary(positions, b, n, x.device)
        x = self.run_layers(x, lambda h, layer: self.attention_many(h, layer, caches, cos, sin))
        if not logits:
            return None
        h = self.rms(x[:, -logits:], self.norm_out)
        return F.linear(h, self.embed).float()

    def forward_device(self, batch, x, logits=0):
        """One frame step of the B requests of `batch` (a RequestBatch whose
        prepare() has run): x [B, n, hidden]. Like forward_many, but every cache
        operation reads the batch's device-resident descriptors, so the whole step
        can be captured once as a CUDA graph and replayed (FrameGraph)."""
        c = self.cfg
        b, n = x.shape[0], x.shape[1]
        cos, sin = self.rotary(batch.positions, b, n, x.device)

        def attend(h, layer):
            q, k, v = self.project_qkv(h, layer, cos, sin)
            out = torch.empty((b, n, c.q_heads, c.head_dim), dtype=q.dtype, device=q.device)
            if batch.append:
                K.append_attention_many_device(q, k, v, batch.targets_ptr, batch.histories_ptr, b, batch.max_past,
                                               out, layer, n, c.kv_heads, c.q_heads // c.kv_heads, c.head_dim,
                                               c.layers)
            else:
                K.packed_attention_many_device(q, k, v, batch.histories_ptr, b, batch.max_past, out, layer, n,
                                               c.kv_heads, c.q_heads // c.kv_heads, c.head_dim, c.layers)
            return self.output(out.reshape(b, n, -1), layer)

        x = self.run_layers(x, attend)
        if not logits:
            return None
        h = self.rms(x[:, -logits:], self.norm_out)
        return F.linear(h, self.embed).float()

    def forward_chunks(self, cache, ids, logits):
        """B equal-length token chunks (ids [B, n]) after the cache's history, side by
        side, without appending; returns fp32 logits [B, logits, vocab] of each
        chunk's last `logits` positions."""
        x = self.embed[ids]
        n = x.shape[1]
        past = cache.get_seq_length(0)
        cos, sin = self.rotary(torch.arange(past, past + n, device=x.device), 1, n, x.device)
        x = self.run_layers(x, lambda h, layer: self.attention_chunks(h, layer, cache, cos, sin))
        h = self.rms(x[:, -logits:], self.norm_out)
        return F.linear(h, self.embed).float()

    def forward(self, cache, ids=None, embeds=None, logits=0):
        """Runs n new tokens (ids [1, n] or embeds [1, n, hidden]) through every layer,
        appending their K/V to `cache`; returns fp32 logits of the last `logits`
        positions (or None)."""
        x = self.embed[ids] if embeds is None else embeds
        n = x.shape[1]
        past = cache.get_seq_length(0)
        cos, sin = self.rotary(torch.arange(past, past + n, device=x.device), 1, n, x.device)
        x = self.run_layers(x, lambda h, layer: self.attention(h, layer, cache, cos, sin))
        if not logits:
            return None
        h = self.rms(x[:, -logits:], self.norm_out)
        return F.linear(h, self.embed).float()


class FrameGraph:
    """Frame steps of B requests replayed from one CUDA graph (the graph-captured
    append of every layer; not in the reference, which launches each layer's
    kernels from Python on every frame). The first step runs eagerly (it is also
    the warm-up); the graph of the whole decoder step is then captured once and
    every later step is: host bookkeeping + one descriptor copy (RequestBatch),
    one input copy, one graph replay. Steps must keep the frame length n; the
    caches' precision may change per step (select() before step()). With
    append=False the steps attend over the caches' histories without appending
    (query chunks side by side, e.g. candidates over one fork)."""

    def __init__(self, model, caches, n, logits=0, max_past=None, append=True):
        self.model, self.n, self.logits = model, n, logits
        self.batch = RequestBatch(caches, n, max_past, append)
        dev = self.batch.device
        self.x = torch.empty((len(caches), n, model.cfg.hidden), dtype=model.embed.dtype, device=dev)
        self.stream = torch.cuda.Stream(dev)
        self.graph = None
        self.out = None

    def rebind(self, caches):
        """Serves another set of caches (same count and geometry) with the same
        captured graph: the next steps append to them."""
        self.batch.rebind(caches)

    def step(self, embeds=None, ids=None):
        """Appends one frame (embeds [B, n, hidden] or ids [B, n]) to every cache;
        returns the logits of the last `logits` positions (None if 0). The returned
        tensor is the graph's output buffer: the next step overwrites it."""
        x = self.model.embed[ids] if embeds is None else embeds
        if tuple(x.shape) != tuple(self.x.shape):
            raise ValueError(f'frame step expects inputs of shape {tuple(self.x.shape)}')
        self.batch.prepare()
        self.x.copy_(x)
        if self.graph is not None:
            self.graph.replay()
            return self.out
        current = torch.cuda.current_stream(self.batch.device)
        self.stream.wait_stream(current)
        with torch.cuda.stream(self.stream):
            out = self.model.forward_device(self.batch, self.x, self.logits)  # the eager first step (warm-up)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=self.stream):
                self.out = self.model.forward_device(self.batch, self.x, self.logits)
        current.wait_stream(self.stream)
        self.graph = graph
        return out
