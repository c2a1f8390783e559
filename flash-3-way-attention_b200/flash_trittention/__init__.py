"""flash_trittention for NVIDIA B200: three-way attention on hand-written sm_100a kernels.

Same public names as the reference package (``src/flash_trittention/__init__.py:11-26``):
``flash_trittention`` (triple-dot-product) and ``TrittentionTriton`` (dot-product-sum),
imported lazily so that ``import flash_trittention`` works without a GPU.
"""

__version__ = "0.1.0"

__all__ = ["flash_trittention", "TrittentionTriton"]  # the reference's public names; the others are extras

_LAZY_ATTRS = {
    "flash_trittention": (".triple_dot_product.flash_trittention", "flash_trittention"),
    "TrittentionTriton": (".dot_product_sum.trittention_triton", "TrittentionTriton"),
    "TrittentionTDP": (".ops", "TrittentionTDP"),  # torch.library operators + module (not in the reference)
    # norms and position rotation of q, k1, k2, in front of either attention
    "qk_norm_rotary": (".norm_rotary", "qk_norm_rotary"),
    "rotary_tables": (".norm_rotary", "rotary_tables"),
    "rotary_axes": (".norm_rotary", "rotary_axes"),
    # serving: a paged cache of quantised rows, and attention of new tokens over it
    "TrittentionCache": (".cache", "TrittentionCache"),
    "new_cache": (".cache", "new_cache"),
    "cache_write": (".cache", "cache_write"),
    "cache_read": (".cache", "cache_read"),
    "tree_ancestors": (".cache", "tree_ancestors"),
    "tdp_decode": (".cache", "tdp_decode"),
    "dps_append": (".cache", "dps_append"),
    "dps_decode": (".cache", "dps_decode"),
    # ... and which of its tokens are kept: the attention weight that each has got, and eviction by it
    "tdp_weigh": (".eviction", "tdp_weigh"),
    "dps_weigh": (".eviction", "dps_weigh"),
    "cache_evict": (".eviction", "cache_evict"),
    # raises if a kernel of an earlier call gave up on a bounded barrier wait (not in the reference)
    "check_status": ("._native", "check_status"),
}


def __getattr__(name):
    try:
        module_path, attr = _LAZY_ATTRS[name]
    except KeyError:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}") from None
    from importlib import import_module

    value = getattr(import_module(module_path, __name__), attr)
    globals()[name] = value
    return value


def __dir__():
    return sorted(list(globals()) + list(_LAZY_ATTRS))
