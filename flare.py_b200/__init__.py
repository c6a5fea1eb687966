"""flare_b200: the FLARE gather-scatter token mixer for NVIDIA B200 (sm_100a).

The directory is named after the project it accelerates (``flare.py_b200``); the
importable name is ``flare_b200`` (see ``flare_b200.py`` at the repository root,
which registers this directory under that name).
"""
from .causal import causal_state_init, flare_causal_decode, flare_causal_mixer, flare_causal_prefill
from .mixer import (device_status, pass_counts, flare_gather, flare_multihead_mixer, flare_scatter, mixer_backward,
                    mixer_forward, set_kernel_path)
from .triple import causal_linear, triple_attention
from .decay import decay_linear, decay_linear_decode, decay_linear_prefill, decay_linear_state_init
from .rotary import Rotary, rotary, rotary_frequencies, rotary_pair
from .modules import FLARE, FLAREBlock, FLAREModel, ResidualMLP
from .cp_train import ContextParallel, ShardedPointCloud, cp_train_step, enable_context_parallel

__all__ = [
    "flare_multihead_mixer", "flare_gather", "flare_scatter", "mixer_forward", "mixer_backward",
    "set_kernel_path", "device_status", "pass_counts", "flare_causal_prefill", "flare_causal_decode", "flare_causal_mixer", "causal_state_init", "triple_attention",
    "causal_linear", "decay_linear", "decay_linear_prefill", "decay_linear_decode", "decay_linear_state_init",
    "rotary", "rotary_pair", "rotary_frequencies", "Rotary", "FLARE", "FLAREBlock", "FLAREModel", "ResidualMLP",
    "ContextParallel", "ShardedPointCloud", "cp_train_step", "enable_context_parallel",
]
