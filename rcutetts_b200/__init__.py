"""rcutetts_b200 -- B200 (sm_100a) per-frame decode path of RCuteTTS.

The compute lives in libcutetts_b200.so (hand-written CUDA behind the C ABI
of include/cutetts_b200.h); this package is the host-side mirror of the
reference crate's model API (see rcutetts_b200.model) and of the paged KV-cache
operators (rcutetts_b200.paged).
"""
import importlib.util as _util
import os as _os

from .config import DiTConfig, FrameConfig, LMConfig, VAEConfig  # noqa: F401

_MODEL_NAMES = {
    "QwenW", "QwenCache", "load_qwen_weights", "prefill", "decode_step", "decode_step_dev",
    "embed_lookup", "DitW", "load_dit_weights", "sway_timesteps", "FrameEngine", "DecoderW",
    "load_decoder_weights", "decode",
}

_PAGED_NAMES = {"PagedStep", "paged_plan", "paged_append", "paged_attention", "paged_attention_workspace"}

# the paged operators need torch and their binding, the rest does not
_HAS_PAGED = _os.path.exists(_os.path.join(_os.path.dirname(__file__), "_paged_ext.so")) and _util.find_spec("torch") is not None

__all__ = ["LMConfig", "DiTConfig", "VAEConfig", "FrameConfig"] + sorted(_MODEL_NAMES | (_PAGED_NAMES if _HAS_PAGED else set()))


def __getattr__(name):
    # Model classes need the CUDA library; import them lazily so config and
    # synth stay importable while the library is being built.
    if name in _MODEL_NAMES:
        from . import model

        return getattr(model, name)
    if name in _PAGED_NAMES:
        from . import paged

        return getattr(paged, name)
    raise AttributeError(name)
