"""
The position rotation's table, for ``MI355XBackend.append_kv_rotated``.

Of a head's elements the first ``rotary_dim`` form pairs, ``(i, i +
rotary_dim / 2)`` or, interleaved, ``(2 i, 2 i + 1)``; at position p pair i
turns by the angle ``p * f[i]``, ``f[i] = theta ** (-2 i / rotary_dim)``
unless the caller gives frequencies of its own (scaled ones, for contexts
longer than a model was trained on). The table holds every position's cosines
and sines, from angles in 64 bits (an angle of 100 000 radians in 32 bits is
off by up to 4e-3), rounded once to 32.
"""

from __future__ import annotations

import torch

__all__ = ["RotaryTable"]


class RotaryTable:
    """
    Cosines and sines of positions ``0 .. max_positions - 1``.

    rotary_dim     elements of a head that turn, even; the rest pass through
    theta          base of the frequencies
    interleaved    pairs are neighbours instead of halves
    frequencies    ``rotary_dim / 2`` angles per position, in place of theta's
    factor         multiplies every cosine and sine (1 for a plain rotation)
    device         where the table lives: the backend's device
    """

    def __init__(self, max_positions: int, rotary_dim: int, *, theta: float = 10000.0,
                 interleaved: bool = False, frequencies=None, factor: float = 1.0,
                 device: str | torch.device = "cuda:0"):
        if max_positions < 1:
            raise ValueError(f"max_positions must be positive, got {max_positions}")
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
        if frequencies is None:
            if not theta > 0:
                raise ValueError(f"theta must be positive, got {theta}")
            f = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64)
                                 / rotary_dim)
        else:
            f = torch.as_tensor(frequencies, dtype=torch.float64).cpu().reshape(-1)
            if f.shape[0] != rotary_dim // 2:
                raise ValueError(f"{f.shape[0]} frequencies given, rotary_dim={rotary_dim} "
                                 f"takes {rotary_dim // 2}")
        self.max_positions, self.rotary_dim = int(max_positions), int(rotary_dim)
        self.interleaved, self.factor = bool(interleaved), float(factor)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        # the stream whose memory the table is; launches on others record it there
        self.stream = (torch.cuda.current_stream(self.device).cuda_stream
                       if self.device.type == "cuda" else None)
        angle = (torch.arange(self.max_positions, dtype=torch.float64, device=self.device)[:, None]
                 * f.to(self.device))
        # [position][cosines, sines][pair]
        self.table = (torch.stack([angle.cos(), angle.sin()], dim=1) * self.factor).float()

    @property
    def cos(self) -> torch.Tensor:
        """(max_positions, rotary_dim / 2), 32 bits."""
        return self.table[:, 0]

    @property
    def sin(self) -> torch.Tensor:
        return self.table[:, 1]

    def __repr__(self) -> str:
        return (f"RotaryTable(max_positions={self.max_positions}, rotary_dim={self.rotary_dim}, "
                f"interleaved={self.interleaved}, device={self.device})")
