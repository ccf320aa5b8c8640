"""Rules of the sources of the kernels around dense latent attention that no run on a GPU can show to hold."""

from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "ascendflow_b200" / "csrc"


def test_shared_sums_are_aligned_as_they_are_accessed():
    """A static shared structure has its members' alignment (8 bytes here) wherever the compiler puts it, unless it asks for more."""
    parts = (CSRC / "latent_parts.cuh").read_text()
    assert "reinterpret_cast<float4*>(&shares.sums" in parts and "struct alignas(16) Shares" in parts


def test_what_kernels_in_front_write_is_read_by_plain_loads():
    """These kernels are resident while the kernel in front still writes what they read behind their wait for it (queries that are turned, rows that are appended, partial sums): the
    read-only path is for memory that nobody writes while a kernel runs."""
    for path in sorted(CSRC.glob("latent_*.cu*")):
        source = path.read_text()
        assert "__ldg(" not in source and "ld.global.nc" not in source and "__restrict__" not in source, path.name
