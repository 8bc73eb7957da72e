"""Models: encoders (``bert``), decoders (``llama``, ``hybrid``), configurations, checkpoints, tokenizers."""


def make_decoder(cfg, device="cuda", seed: int = 0, tp=None, weights: dict | None = None, dtype: str = "bf16",
                 kv_bits: int = 16, kv_keep: int = 0, kv_recent: int = 0):
    """The decoder of a configuration: its checkpoint's weights if it names a folder, else seeded random ones. kv_bits, kv_keep,
    kv_recent: the cache of Llama / Phi-3 decoders (``LlamaDecoder``)."""
    from .configs import HybridConfig, decoder_dtypes
    if dtype not in decoder_dtypes(cfg):
        raise ValueError(f"{cfg.name}: dtype {dtype!r} is not supported ({', '.join(decoder_dtypes(cfg))})")
    if isinstance(cfg, HybridConfig):
        from .hybrid import HybridDecoder
        if kv_bits != 16 or kv_keep or kv_recent:
            raise ValueError(f"{cfg.name}: its caches are in the activations' type (kv_bits=16, kv_keep=0, kv_recent=0)")
        return HybridDecoder(cfg, device, seed=seed, tp=tp, weights=weights, dtype=dtype)
    from .llama import LlamaDecoder
    return LlamaDecoder(cfg, device, seed=seed, tp=tp, weights=weights, kv_bits=kv_bits, kv_keep=kv_keep, kv_recent=kv_recent)
