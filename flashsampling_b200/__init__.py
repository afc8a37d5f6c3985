"""B200-native fused LM-head sampling (matmul + Gumbel-max in one pass over the weight), and beam search beside it."""

from .beam import BeamSearch, BeamStep, beam_search_step, reorder_beams  # noqa: F401
from .core import (  # noqa: F401
    PROVIDERS,
    PreparedSampler,
    Sampler,
    SimpleSampler,
    check_status,
    fused_mm_sample,
    fused_mm_sample_triton,
    get_sampler,
    last_path,
)
from .int4 import Int4Weight, int4_linear  # noqa: F401
from .tp_info import TP1, TPInfo, run_maybe_distributed  # noqa: F401

__version__ = "0.1.0"
