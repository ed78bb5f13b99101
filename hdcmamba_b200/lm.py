"""Language-model wrapper and the benchmark configurations.

The reference keeps its LM wrappers outside the package (train.py:116-151,
train_fineweb.py:23-94): token embedding -> HdcMamba backbone -> LayerNorm ->
lm_head tied to the embedding.  ``HdcMambaLM`` is that wrapper; the head is
``F.linear(h, embedding.weight)`` so that no extra Linear is constructed (an
extra module would consume RNG and change seeded weights).

``build_lm(cfg)`` creates the seeded synthetic-weight models of the benchmark
configurations: seed 0, every Linear/Conv1d/Embedding weight re-drawn
N(0, 0.02) in ``named_parameters`` order, norms at gamma=1 / beta=0, biases,
A_log, decay_log and gamma_buf at the reference's own init.
"""
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .model import HdcMamba9v3Block, HdcMamba9v3Model, final_layer_norm
from .training import embedding


_forward = nn.Embedding.forward


def embed(module, ids):
    """``module(ids)``: through the framework's lookup for an ``nn.Embedding`` as it comes (no renormalised
    rows, sparse or frequency-scaled gradients, and nothing that would see or change the module's call), in
    fp32 or bf16; otherwise the module itself."""
    if type(module) is nn.Embedding and _is_plain(module, ids) and not _is_watched(module):
        return embedding(ids, module.weight, padding_idx=module.padding_idx)
    return module(ids)


def _is_plain(module, ids):
    """The module does what the lookup does, with a table and ids that the lookup takes."""
    return (module.max_norm is None and not module.scale_grad_by_freq and not module.sparse
            and _lib.host().embedding_takes(ids, module.weight))


def _is_watched(module):
    """Hooks of the module or of all modules, a forward that is not the class's own (offloading, adapters,
    ``module.compile()``), modes that see every operation."""
    return (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks
            or nn.modules.module._has_any_global_hook() or "forward" in module.__dict__ or nn.Embedding.forward is not _forward
            or module._compiled_call_impl is not None or torch._C._len_torch_function_stack() or torch._C._len_torch_dispatch_stack())


class HdcMambaLM(nn.Module):
    """Embedding -> blocks (or HdcMamba9v3Model) -> LayerNorm -> tied head."""

    def __init__(self, vocab_size, d_model, n_layers, d_state, num_heads, chunk_size=256, use_model=True,
                 semantics="fixed"):
        super().__init__()
        self.use_model = use_model
        self.embedding = nn.Embedding(vocab_size, d_model)
        if use_model:
            self.backbone = HdcMamba9v3Model(d_model, n_layers, d_state, num_slots=32, num_heads=num_heads,
                                             semantics=semantics)
        else:
            self.layers = nn.ModuleList([HdcMamba9v3Block(d_model=d_model, d_state=d_state, num_heads=num_heads,
                                                          chunk_size=chunk_size, semantics=semantics)
                                         for _ in range(n_layers)])
        self.norm = nn.LayerNorm(d_model)

    def hidden(self, ids):
        h = embed(self.embedding, ids)  # a fresh activation: the layers update it in place
        if self.use_model:
            return self.backbone._forward(h, owns_input=True)
        for layer in self.layers:
            h = layer._forward_inplace(h)
        return h

    def forward(self, ids):
        return F.linear(final_layer_norm(self.norm, self.hidden(ids)), self.embedding.weight)


@dataclass(frozen=True)
class LMConfig:
    name: str
    vocab: int
    d_model: int
    n_layers: int
    d_state: int
    num_heads: int
    chunk_size: int
    use_model: bool
    batch: int
    seq_len: int


CONFIGS = {
    # the reference's CPU-runnable plumbing case (fp32)
    "c1": LMConfig("c1", 4096, 256, 2, 64, 8, 64, False, 1, 512),
    # 24 x d1024, H16, ds128 (train_fineweb.py:38), chunk 256 (model.py:399)
    "c4": LMConfig("c4", 50304, 1024, 24, 128, 16, 256, True, 8, 4096),
    # 12 x d768, H12, ds64 (train_fineweb.py:33), chunk 256, B1 x L32768
    "c5": LMConfig("c5", 50304, 768, 12, 64, 12, 256, True, 1, 32768),
}


def reinit_(module, std=0.02):
    """Re-draw every Linear / Conv1d / Embedding weight N(0, std) in named_parameters order."""
    mods = dict(module.named_modules())
    with torch.no_grad():
        for name, p in module.named_parameters():
            owner = mods[name.rsplit(".", 1)[0]] if "." in name else module
            if name.endswith("weight") and isinstance(owner, (nn.Linear, nn.Conv1d, nn.Embedding)):
                p.normal_(0.0, std)
    return module


def build_lm(cfg, seed=0, semantics="fixed"):
    """Seeded synthetic-weight LM for a config (constructed on CPU, fp32)."""
    if isinstance(cfg, str):
        cfg = CONFIGS[cfg]
    torch.manual_seed(seed)
    lm = HdcMambaLM(cfg.vocab, cfg.d_model, cfg.n_layers, cfg.d_state, cfg.num_heads, cfg.chunk_size,
                    cfg.use_model, semantics=semantics)
    return reinit_(lm).eval()


def synthetic_ids(cfg, seed=0, batch=None, seq_len=None):
    """Uniform token ids [B, L] from a dedicated generator."""
    if isinstance(cfg, str):
        cfg = CONFIGS[cfg]
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, cfg.vocab, (batch or cfg.batch, seq_len or cfg.seq_len), generator=g)
