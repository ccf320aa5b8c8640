"""Rules of the sources of the kernels around dense latent attention that no run on a GPU can show to hold."""

from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "ascendflow_b200" / "csrc"


def test_shared_sums_are_aligned_as_they_are_accessed():
    """A static shared structure has its members' alignment (8 bytes here) wherever the compiler puts it, unless it asks for more."""
    parts = (CSRC / "latent_parts.cuh").read_text()
    assert "reinterpret_cast<float4*>(&shares.sums" in parts and "struct alignas(16) Shares" in parts
