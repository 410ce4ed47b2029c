"""RoPE cos/sin tables (host, built once at load).

Same construction as the reference's RoPECacheBuilder.build_cache
(vte/compiler/rope_cache_builder.py:42-97): freq_i = 1 / theta^(i / (hd/2))
in fp32, angle = pos * freq_i, cos/sin rounded to fp16 and duplicated into
both halves of a [max_seq, head_dim] table ("rotate-half" layout read by
rope_kernel at [pos * head_dim + i]).
"""
from __future__ import annotations

import numpy as np


def build_rope_cache(max_seq_len: int, head_dim: int, rope_theta: float) -> tuple[np.ndarray, np.ndarray]:
    half = head_dim // 2
    freqs = 1.0 / (np.float32(rope_theta) ** (np.arange(0, half, dtype=np.float32) / np.float32(half)))
    angles = np.outer(np.arange(max_seq_len, dtype=np.float32), freqs.astype(np.float32))
    cos_h = np.cos(angles).astype(np.float16)
    sin_h = np.sin(angles).astype(np.float16)
    return np.ascontiguousarray(np.concatenate([cos_h, cos_h], 1)), np.ascontiguousarray(np.concatenate([sin_h, sin_h], 1))


def rope_frequencies(rotary_dim: int, rope_theta: float, scaling: str | None = None, factor: float = 1.0,
                     original_context: int = 0, fast: float = 32.0, slow: float = 1.0,
                     amplitude: float | None = None) -> tuple[np.ndarray, float]:
    """Radians per position of each of the rotary_dim / 2 pairs (float64), and the amplitude of a ``HeadForm``.

    freq_i = rope_theta^(-2 i / rotary_dim), scaled for contexts ``factor`` times as long:
      * "linear": all of them divided by ``factor``;
      * "base": the base times factor^(r / (r - 2)) with r = rotary_dim (so the slowest pair is divided by ``factor``, the
        fastest stays);
      * "turns": pairs that turn ``fast`` times or more in ``original_context`` positions stay, those that turn ``slow``
        times or less are divided by ``factor``, in between linearly in the number of turns; amplitude 1;
      * "yarn": the same with a ramp that is linear in the pair's index, between the whole pairs around where pairs turn
        ``fast`` and ``slow`` times, and an amplitude of 0.1 ln(factor) + 1 (Peng et al. 2023, "YaRN: Efficient Context
        Window Extension of Large Language Models").
    ``amplitude`` overrides the form's own."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} is not an even number from 2 on")
    if not rope_theta > 0 or not factor > 0:
        raise ValueError("rope_theta and factor must be above 0")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    freq = float(rope_theta) ** (-2 * i / rotary_dim)
    own = 1.0
    if scaling is None:
        pass
    elif scaling == "linear":
        freq = freq / factor
    elif scaling == "base":
        if rotary_dim < 4:
            raise ValueError("scaling the base needs two pairs")
        freq = (float(rope_theta) * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim)
    elif scaling in ("turns", "yarn"):
        if original_context < 1 or not fast > slow > 0:
            raise ValueError(f"{scaling}: original_context from 1 on and fast > slow > 0 are needed")
        if scaling == "turns":
            stays = np.clip((original_context * freq / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        else:
            if not rope_theta > 1:
                raise ValueError("yarn: rope_theta above 1 is needed")

            def pair(turns):
                return rotary_dim * np.log(original_context / (turns * 2 * np.pi)) / (2 * np.log(rope_theta))
            low, high = max(np.floor(pair(fast)), 0.0), min(np.ceil(pair(slow)), rotary_dim - 1.0)
            stays = 1 - np.clip((i - low) / max(high - low, 1e-3), 0, 1)
            own = 0.1 * float(np.log(factor)) + 1 if factor > 1 else 1.0
        freq = freq * (stays + (1 - stays) / factor)
    else:
        raise ValueError(f"unknown scaling {scaling!r}")
    return freq, own if amplitude is None else float(amplitude)
