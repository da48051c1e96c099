"""The package's version, which users of the reference read as `__version__` (reference
mlx_recurrence/__init__.py:90): the version it follows and the target."""
import mlx_recurrence_amd as mr


def test_version():
    assert mr.__version__ == "0.3.0+gfx950"
