"""The half-width RoPE tables are kept per rope object, not per address."""

from __future__ import annotations

import torch

from deltakv_b200.rope import RotaryEmbedding, half_tables

CPU = torch.device("cpu")


def test_tables_of_a_new_rope_are_its_own():
    """Objects and tensors made and dropped in turn reuse addresses; the tables must not."""
    for i in range(200):
        hd, base = (64, 128, 32)[i % 3], 10000.0 + i
        rope = RotaryEmbedding(hd, 50, base)
        cos, sin = half_tables(rope, CPU)
        assert cos.shape == (50, hd // 2)
        assert torch.equal(cos, rope.cos_cached[:, : hd // 2]) and torch.equal(sin, rope.sin_cached[:, : hd // 2])
        del rope


def test_tables_follow_a_changed_rope():
    rope = RotaryEmbedding(64, 50)
    first = half_tables(rope, CPU)
    assert half_tables(rope, CPU)[0] is first[0]
    rope.cos_cached.mul_(0.5)  # rescaled in place
    assert torch.equal(half_tables(rope, CPU)[0], rope.cos_cached[:, :32])
    longer = RotaryEmbedding(64, 90)
    rope.cos_cached, rope.sin_cached = longer.cos_cached, longer.sin_cached
    assert half_tables(rope, CPU)[0].shape == (90, 32)


def test_tables_from_a_module_and_inference_mode():
    class Rope(torch.nn.Module):
        def __init__(self):
            super().__init__()
            r = RotaryEmbedding(16, 9)
            self.register_buffer("cos_cached", r.cos_cached)
            self.register_buffer("sin_cached", r.sin_cached)

    with torch.inference_mode():
        rope = Rope()
        assert half_tables(rope, CPU)[0].shape == (9, 8)
    assert half_tables(rope, CPU)[1].shape == (9, 8)


def test_tables_follow_a_rope_changed_in_inference_mode():
    """Tensors of inference mode have no version; ordinary ones count changes made in it."""
    with torch.inference_mode():
        rope = RotaryEmbedding(64, 50)
        bare = RotaryEmbedding(64, 50)
        bare.cos_cached, bare.sin_cached = bare.cos_cached.clone(), bare.sin_cached.clone()
        assert bare.cos_cached.is_inference() and not rope.cos_cached.is_inference()
        for r in (rope, bare):
            half_tables(r, CPU)
            r.cos_cached.mul_(0.5)
            assert torch.equal(half_tables(r, CPU)[0], r.cos_cached[:, :32])
    assert half_tables(rope, CPU)[0] is half_tables(rope, CPU)[0]
    assert torch.equal(half_tables(bare, CPU)[0], bare.cos_cached[:, :32])


def test_tables_of_a_rope_that_cannot_be_kept():
    class Bare:
        __slots__ = ("cos_cached", "sin_cached")  # no weak references

    rope, source = Bare(), RotaryEmbedding(64, 50)
    rope.cos_cached, rope.sin_cached = source.cos_cached, source.sin_cached
    for _ in range(2):
        cos, sin = half_tables(rope, CPU)
        assert torch.equal(cos, source.cos_cached[:, :32]) and torch.equal(sin, source.sin_cached[:, :32])
        rope.cos_cached.mul_(0.5)
