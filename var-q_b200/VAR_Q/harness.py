"""A stand-in for the model loop around the hook, for whole-loop throughput numbers.

The reference measures generation through ``VAR.autoregressive_infer_cfg`` (VAR/models/var.py:130-193): CFG doubles the
batch, ``kv_caching(True)`` is switched on in every block, and for each scale of the schedule the new token map runs
through all blocks, each of which projects QKV, takes the hook (quantize + cache + attention) and applies its MLP.
The reference's model classes, tokenizer and checkpoints do not travel with this package, so ``StandInVAR`` rebuilds
only that skeleton with randomly initialised torch layers of the same shapes: LayerNorm -> attention (with
``VAR_Q.hooks.install``) -> LayerNorm -> 4x MLP per block, a random token map per scale in place of sampling and
embedding.  It exists to time the hot path where it runs in practice -- between GEMMs, launched from Python or
replayed as one CUDA graph -- not to generate images.

``StandInDecoder`` is the same for serving: a causal decoder skeleton over paged caches, whose sequences come, are prefilled chunk by chunk next to
others that decode token by token, and go.
"""
import math
from typing import Optional, Sequence

import torch

from .hooks import install
from .paged import PagedCache, PageTable


class StandInSelfAttention(torch.nn.Module):
    """Carries the attributes ``hooks.install`` reads (the reference class's, VAR/models/basic_var.py:73-117)."""

    def __init__(self, width: int, heads: int, block_idx: int, q_bits: int, quant_method: str, attn_l2_norm: bool = True):
        super().__init__()
        self.block_idx, self.num_heads, self.head_dim = block_idx, heads, width // heads
        self.attn_l2_norm, self.q_bits, self.quant_method, self.qkv_format = attn_l2_norm, q_bits, quant_method, 'BLHc'
        self.enable_quantization = True
        if attn_l2_norm:
            self.scale = 1
            self.scale_mul_1H11 = torch.nn.Parameter(torch.full((1, heads, 1, 1), 4.0).log())
            self.max_scale_mul = math.log(100)
        else:
            self.scale = 0.25 / math.sqrt(self.head_dim)
        self.mat_qkv = torch.nn.Linear(width, 3 * width, bias=False)
        self.q_bias, self.v_bias = torch.nn.Parameter(torch.zeros(width)), torch.nn.Parameter(torch.zeros(width))
        self.register_buffer('zero_k_bias', torch.zeros(width))
        self.proj, self.proj_drop = torch.nn.Linear(width, width), torch.nn.Identity()
        self.caching, self.k_quant, self.v_quant = False, None, None

    def kv_caching(self, enable: bool):
        self.caching = enable
        self.k_quant = self.v_quant = None

    def forward(self, x, attn_bias=None):
        raise RuntimeError("StandInSelfAttention only runs with kv_caching(True) and the installed packed-cache route")


class StandInBlock(torch.nn.Module):
    def __init__(self, width, heads, block_idx, q_bits, quant_method, max_tokens, k_kwargs, v_kwargs):
        super().__init__()
        self.ln1, self.ln2 = torch.nn.LayerNorm(width), torch.nn.LayerNorm(width)
        self.attn = install(StandInSelfAttention(width, heads, block_idx, q_bits, quant_method), max_tokens, k_kwargs, v_kwargs)
        self.fc1, self.fc2 = torch.nn.Linear(width, 4 * width), torch.nn.Linear(4 * width, width)

    def forward(self, x):
        x = x + self.attn(self.ln1(x), None)
        return x + self.fc2(torch.nn.functional.gelu(self.fc1(self.ln2(x)), approximate='tanh'))


class StandInVAR(torch.nn.Module):
    def __init__(self, depth: int = 16, width: int = 1024, heads: int = 16,
                 patch_nums: Sequence[int] = (1, 2, 3, 4, 5, 6, 8, 10, 13, 16), q_bits: int = 8,
                 quant_method: str = 'G_TOKEN_HEAD', k_kwargs: Optional[dict] = None, v_kwargs: Optional[dict] = None):
        super().__init__()
        self.width, self.patch_nums = width, tuple(patch_nums)
        total = sum(p * p for p in patch_nums)
        self.blocks = torch.nn.ModuleList(StandInBlock(width, heads, i, q_bits, quant_method, total, k_kwargs, v_kwargs)
                                          for i in range(depth))

    @torch.inference_mode()
    def generate(self, token_maps: Sequence[torch.Tensor]) -> torch.Tensor:
        """One pass over the scale schedule.  ``token_maps[i]`` is the (CFG-doubled) input of scale i, [2B, pn_i^2, width];
        returns the last scale's hidden state."""
        for b in self.blocks:
            b.attn.kv_caching(True)
        x = None
        for tm in token_maps:
            x = tm
            for b in self.blocks:
                x = b(x)
        for b in self.blocks:
            b.attn.kv_caching(False)
        return x

    def token_maps(self, batch: int, device, dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)
        return [torch.randn((2 * batch, p * p, self.width), generator=g, device=device, dtype=torch.float32).to(dtype)
                for p in self.patch_nums]


class StandInDecoderBlock(torch.nn.Module):
    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int, cache: PagedCache, window: Optional[int], sinks: int):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.cache, self.window, self.sinks = heads, kv_heads, head_dim, cache, window, sinks
        self.ln1, self.ln2 = torch.nn.LayerNorm(width), torch.nn.LayerNorm(width)
        self.qkv = torch.nn.Linear(width, (heads + 2 * kv_heads) * head_dim, bias=False)
        self.proj = torch.nn.Linear(heads * head_dim, width, bias=False)
        self.fc1, self.fc2 = torch.nn.Linear(width, 4 * width), torch.nn.Linear(4 * width, width)

    def forward(self, x, slots, batch):
        # q, k and v stay views of the fused activation: the operators read them with their strides
        q, k, v = self.qkv(self.ln1(x)).unflatten(-1, (-1, self.head_dim)).split((self.heads, self.kv_heads, self.kv_heads), 1)
        self.cache.append(k, v, slots)
        out = self.cache.attend(q, *batch, 1.0 / math.sqrt(self.head_dim), window=self.window, sinks=self.sinks)
        x = x + self.proj(out.flatten(1))
        return x + self.fc2(torch.nn.functional.gelu(self.fc1(self.ln2(x)), approximate='tanh'))


class StandInDecoder(torch.nn.Module):
    """``step`` advances any mix of sequences by any number of tokens each; one ``PageTable`` serves all layers, each of which has a cache of its own."""

    def __init__(self, depth: int = 4, width: int = 1024, heads: int = 16, kv_heads: int = 4, head_dim: int = 64, num_pages: int = 256, page_size: int = 64,
                 k_bits: int = 8, v_bits: int = 8, window: Optional[int] = None, sinks: int = 0, device="cuda"):
        super().__init__()
        self.table, self.device_ = PageTable(num_pages, page_size), device
        caches = [PagedCache(num_pages, page_size, kv_heads, head_dim, k_bits, v_bits, device) for _ in range(depth)]
        self.blocks = torch.nn.ModuleList(StandInDecoderBlock(width, heads, kv_heads, head_dim, c, window, sinks) for c in caches)
        self.to(device)

    @torch.inference_mode()
    def step(self, seqs: Sequence, xs: Sequence[torch.Tensor]) -> Sequence[torch.Tensor]:
        """``xs[i]`` ``[n_i, width]``: the next inputs of ``seqs[i]`` (new sequences are taken in).  Returns their hidden states."""
        new, counts = [s for s in dict.fromkeys(seqs) if s not in self.table], [x.size(0) for x in xs]
        for s in new:
            self.table.add(s)
        try:
            slots = self.table.extend(seqs, counts, self.device_)
        except Exception:
            for s in new:
                self.table.remove(s)
            raise
        batch = self.table.batch(seqs, counts, self.device_)
        x = torch.cat(list(xs))
        for b in self.blocks:
            x = b(x, slots, batch)
        return x.split(counts)

    def finish(self, seq) -> None:
        self.table.remove(seq)
