"""How attention of single tokens over pages of 8 bits cuts the keys: choices that do not jump between sizes next to each other, and measured ones."""
import pytest

from ghost_flow_b200.ops.paged import _parts_of_8_bits


@pytest.mark.parametrize("kv_heads", [1, 2, 8, 12, 32])
def test_sizes_next_to_each_other(kv_heads):
    """Where a choice changes, both are near the best: it never goes between few parts and 16 while CTAs fill the machine."""
    for B in (1, 2, 3, 5, 8, 13, 16, 24, 30, 31, 32, 33, 40, 64, 96, 160):
        for keys in range(64, 12000, 64):
            a, units = _parts_of_8_bits(B * kv_heads, keys, 148, kv_heads), keys // 64
            assert a == -(592 // kv_heads) or 1 <= a <= min(16, units)
            if a > 1:
                assert B * kv_heads * (a - 1) <= 3 * 592               # one part less would do where the machine is full three times
            if a < 0:
                assert B * kv_heads * units >= 20 * 592


# us by parts, uniform lengths, 148 SMs: (sequences, KV heads, keys at most, D) -> the choices within a quarter of the best
@pytest.mark.parametrize("B,kv_heads,keys,good", [
    (96, 8, 2048, (1, 2, 3, 4, -74)),              # 47 / 51 / 53 / 57 / 51; 16 parts 107
    (40, 8, 2048, (1, 2, 3, 4, 5, -74)),           # 27 / 29 / 29 / 30 / 31 / 29; 16 parts 52
    (31, 8, 4096, (2, 3, 4, 5, 8, -74)),           # 44 / 37 / 39 / 39 / 41 / 38; 16 parts 55
    (31, 8, 4032, (2, 3, 4, 5, 8, -74)),
    (40, 32, 2048, (1, 2, 3, 4, -18)),             # 68 / 68 / 71 / 76 / 65; 16 parts 140
    (96, 32, 512, (1, -18)),                       # 49 / 60; 4 parts 94
    (96, 8, 1024, (1, 2)),                         # 31 / 38; 8 parts 61
    (24, 32, 1024, (1, 2, 3, -18)),                # 29 / 31 / 34 / 33; 8 parts 50
    (2, 8, 8000, (8, 16)),                         # 12 / 12; 4 parts 16
    (1, 8, 8000, (8, 16)),
])
def test_measured_choices(B, kv_heads, keys, good):
    assert _parts_of_8_bits(B * kv_heads, keys, 148, kv_heads) in good
