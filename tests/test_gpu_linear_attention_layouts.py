"""Linear attention in every layout of its scans: padded head dimension (16, 32, 64, 96, 128) x
columns of a wavefront (8, 16, 32) x aligned operands or not, forward and backward, with and
without the time axis split.

How many columns a wavefront takes follows from the number of heads: 32 where
B H ceil(D / 32) reaches 2048 (backward 1024; forward 1536 for 65 to 96 features), 16 where half
of that suffices, else 8 (16 above 64 features). From 128 tokens on chunks of 32 tokens or more
make up for heads, so that the split cases need a quarter of them. Odd head dimensions read
their operands a value at a time, multiples of four 16 bytes.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_sequence_accuracy import check_by_age

pytestmark = pytest.mark.gpu

# (B, T, H, D)  # padded head dimension: columns forward, backward; chunks forward, backward
UNSPLIT = [
    (64, 19, 2, 13),    # 16: 8, 8
    (512, 19, 2, 13),   # 16: 8, 16
    (1024, 19, 2, 13),  # 16: 16, 16
    (128, 27, 2, 12),   # 16: 8, 8
    (1024, 19, 2, 16),  # 16: 16, 16
    (33, 27, 2, 27),    # 32: 8, 8
    (64, 27, 8, 27),    # 32: 8, 16
    (512, 27, 2, 27),   # 32: 16, 32
    (512, 19, 4, 27),   # 32: 32, 32
    (33, 27, 2, 20),    # 32: 8, 8
    (64, 27, 8, 20),    # 32: 8, 16
    (512, 27, 2, 20),   # 32: 16, 32
    (512, 19, 4, 20),   # 32: 32, 32
    (16, 19, 2, 57),    # 64: 8, 8
    (33, 27, 8, 57),    # 64: 8, 16
    (64, 19, 8, 57),    # 64: 16, 32
    (128, 19, 8, 61),   # 64: 32, 32
    (16, 19, 2, 40),    # 64: 8, 8
    (171, 27, 2, 40),   # 64: 8, 16
    (128, 27, 3, 40),   # 64: 8, 16
    (64, 19, 8, 40),    # 64: 8, 32
    (128, 19, 8, 40),   # 64: 32, 32
    (64, 19, 4, 90),    # 96: 16, 16
    (64, 19, 8, 90),    # 96: 32, 32
    (64, 19, 4, 72),    # 96: 16, 16
    (64, 19, 8, 72),    # 96: 32, 32
    (33, 19, 4, 125),   # 128: 16, 16
    (64, 19, 8, 125),   # 128: 32, 32
    (33, 19, 4, 100),   # 128: 16, 16
    (64, 19, 8, 100),   # 128: 32, 32
]
SPLIT = [
    (16, 130, 8, 13),   # 16: 8, 16; 4, 4
    (64, 130, 8, 13),   # 16: 16, 16; 4, 2
    (16, 130, 4, 27),   # 32: 8, 16; 4, 4
    (16, 130, 4, 20),   # 32: 8, 16; 4, 4
    (64, 130, 4, 20),   # 32: 16, 32; 4, 4
    (64, 130, 4, 27),   # 32: 16, 32; 4, 4
    (16, 130, 2, 57),   # 64: 8, 16; 4, 4
    (16, 130, 3, 40),   # 64: 8, 16; 4, 4
    (16, 130, 8, 57),   # 64: 16, 32; 4, 4
    (171, 130, 1, 40),  # 64: 16, 32; 4, 3
    (5, 1030, 8, 57),   # 64: 32, 32; 26, 13
    (16, 130, 8, 90),   # 96: 32, 32; 4, 2
    (16, 300, 8, 125),  # 128: 32, 16; 4, 1
    (1, 700, 3, 100),   # 128: 16, 16; 18, 18
]


@pytest.mark.parametrize("B,T,H,D", UNSPLIT + SPLIT)
def test_layout(dev, B, T, H, D):
    decay = torch.tensor([0.97, 0.0, 1.0, 0.1, 0.5, 0.999, 0.26, 0.9])[torch.arange(H) % 8]
    lengths = None
    if B % 2 == 0:  # ragged, with lengths at the ends
        lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B + D))
        lengths[:2] = torch.tensor([0, T])
    check_by_age(dev, B, T, H, D, decay, lengths=lengths, state=H % 4 == 0, seed=D)
