"""What asks for the canonical replay cannot get it behind a shared prefix, and is told so."""
import pytest
import torch

from adkv_b200.cache import KVCache, KVCacheLayer
from adkv_b200.e2e_llama import ADKVLlama, LlamaShape


def _filled(layer):
    """A layer as it is after a prefill of three tokens, in host memory: what fork looks at before anything else."""
    layer._bind(1, 2, 128, torch.device("cpu"))
    layer._reserve(3)
    layer._n = 3
    return layer


def test_the_canonical_replay_is_refused_behind_a_prefix():
    with pytest.raises(ValueError, match="fast=False"):
        _filled(KVCacheLayer(fast=False)).fork(2)
    caches = KVCache(2, fast=False)
    for c in caches:
        _filled(c)
    with pytest.raises(ValueError, match="fast=False"):
        caches.fork(2)
    for fast in (None, True):
        with pytest.raises(RuntimeError, match="CUDA"):          # as far as the tensors
            _filled(KVCacheLayer(fast=fast)).fork(2)
    shape = LlamaShape(n_layers=0, d_model=32, n_heads=2, n_kv_heads=2, head_dim=128, ffn=64, vocab=50)
    with pytest.raises(ValueError, match="fast=False"):
        ADKVLlama(shape, 2, 8, device="cpu", shared_tokens=8, fast=False)
    for fast in (None, True):
        assert ADKVLlama(shape, 2, 8, device="cpu", shared_tokens=8, fast=fast).fast
    assert not ADKVLlama(shape, 2, 8, device="cpu", fast=False).fast
