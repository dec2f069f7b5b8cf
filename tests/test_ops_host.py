"""CPU tests of the paged-cache operators' host side: exported symbols,
argument layouts, refusals that need no device, and the rotary tables."""
import ctypes as C
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest

from lrrt_b200 import native as N

REPO = Path(__file__).resolve().parents[1]


def test_operators_library_exports_every_declared_symbol(built):
    text = (REPO / "include" / "lrrt_ops.h").read_text()
    names = sorted(set(re.findall(r"LRRT_API\s+[\w\s\*]+?\b(lro_\w+)\s*\(", text)))
    assert names == sorted(N.OPS_FUNCTIONS)
    for name in names:
        assert hasattr(N.operators(), name), name
    assert hasattr(N.runtime(), "lr_queue_wrap_stream")


def test_host_checks_and_struct_sizes(built):
    result = subprocess.run([str(built["test:ops_host_test"])], capture_output=True, text=True,
                            timeout=120)
    assert result.returncode == 0, result.stderr
    assert "ops host checks: ok" in result.stdout
    sizes = dict(zip(*[iter(result.stdout.split("sizes:")[1].split("\n")[0].split())] * 2))
    for name, struct in (("rope_append", N.RopeAppend), ("paged_attention", N.PagedAttention),
                         ("fork", N.PagesFork), ("compact", N.PagesCompact),
                         ("copy", N.PagesCopy), ("beam", N.BeamSelect)):
        assert C.sizeof(struct) == int(sizes[name]), name


@pytest.mark.parametrize("rotary,theta,scaling", [
    (64, 1e6, {}), (2, 1e4, {}), (48, 5e5, dict(factor=4.0)),
    (128, 1e6, dict(factor=8.0, low_turns=1.0, high_turns=4.0, trained_positions=8192)),
    (64, 1e4, dict(factor=2.0, low_turns=2.0, high_turns=2.0, trained_positions=4096)),
])
def test_rope_tables(built, rotary, theta, scaling):
    """Against extended precision: one rounding to 32 bits, and an angle of
    p * f in 64 bits, off by at most 3 * 2^-53 of itself."""
    from lrrt_b200 import ops
    positions = 5000
    cos, sin = ops.rope_tables(positions, rotary, theta, **scaling)
    i = np.arange(rotary // 2, dtype=np.longdouble)
    f = np.longdouble(theta) ** (-2 * i / rotary)
    factor = scaling.get("factor", 1.0)
    if factor > 1:
        low, high = scaling.get("low_turns", 0.0), scaling.get("high_turns", 0.0)
        keep = np.zeros_like(f)
        if high > 0:
            turns = scaling["trained_positions"] * f / (2 * np.pi)
            keep = np.clip((turns - low) / (high - low), 0, 1) if high > low else \
                (turns >= high).astype(np.longdouble)
        f = f * keep + f / factor * (1 - keep)
    angle = np.arange(positions, dtype=np.longdouble)[:, None] * f
    bound = 2.0 ** -25 + positions * 8 * 2.0 ** -53
    assert np.abs(cos - np.cos(angle)).max() <= bound
    assert np.abs(sin - np.sin(angle)).max() <= bound


def test_rope_tables_refuse(built):
    from lrrt_b200 import ops
    with pytest.raises(N.LrrtError, match="rotary_dim"):
        ops.rope_tables(4, 7)
    with pytest.raises(N.LrrtError, match="factor"):
        ops.rope_tables(4, 8, factor=0.0)
