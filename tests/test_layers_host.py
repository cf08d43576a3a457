"""The host's part of the layer operators: loading, binding, and what is refused there (no GPU needed)."""
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_every_lane_of_a_row_holds_the_same_sum():
    """The lane exchanges of layers.hpp's group_sum, replayed: partners exchange, so both add the same two numbers and addition's order is no matter."""
    import re

    import numpy as np
    text = (ROOT / "vmc_pde_amd" / "csrc" / "layers.hpp").read_text()
    body = text[text.index("A group_sum(A v)"):text.index("// elements of a 16-byte vector")]
    steps = [int(v, 16) for v in re.findall(r"dpp_move<(0x[0-9a-f]+)>", body)]
    assert len(steps) == 4

    def source(control, lane):
        row, i = lane & ~15, lane & 15
        if control < 0x100:                                    # quad_perm
            return row | (i & ~3) | (control >> 2 * (i & 3) & 3)
        if 0x121 <= control <= 0x12f:                          # row_ror
            return row | (i - (control & 15)) % 16
        return row | {0x140: 15 - i, 0x141: (i & 8) | 7 - (i & 7)}[control]
    v = np.random.default_rng(1).standard_normal((1000, 64)).astype(np.float32)
    for control in steps:
        v = v + v[:, [source(control, lane) for lane in range(64)]]
    rows = v.reshape(1000, 4, 16)
    assert (rows == rows[:, :, :1]).all()
