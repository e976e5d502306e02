"""B200-native SemanticLogKV flush-and-attend path (sm_100a CUDA behind a C-ABI library)."""
from .attention import log_kv_chunk_attention, log_kv_shared_attention, log_kv_tree_attention, pack_mid_kv  # noqa: F401
from .cache import LogStructuredKVCache, _SemanticReplayUpdates  # noqa: F401
from .beam import beam_select  # noqa: F401
from .logits import adjust_logits  # noqa: F401
from .rotary import log_kv_rotate, scaled_rope_tables  # noqa: F401
