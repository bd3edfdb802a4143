"""Long-cache operators without a GPU: a null context is refused by every entry point."""
import gpullama_attn as gla


def test_null_context_is_refused():
    L = gla.lib()
    for t in ("f32kv", "f16kv"):
        for name in (f"gla_block_bounds_{t}", f"gla_rope_append_batched_{t}", f"gla_block_select_{t}",
                     f"gla_decode_blocks_{t}", f"gla_decode_weights_{t}", f"gla_kv_evict_{t}"):
            fn = getattr(L, name)
            args = [None if a is gla._P else 0 for a in fn.argtypes]
            assert fn(*args) == -1, name
