"""Register spills of the kernels between an attention block's projections, from the metadata in libdramamoe.so (CPU)."""
import pytest

from test_kernel_registers import READELF, _spills

# Kept in memory in part, as the comment beside it says: tiles of heads above 192 elements.
SPILL = "k_attn_tilesILi8E"


@pytest.mark.skipif(READELF is None, reason="no llvm-readelf")
def test_spills(tmp_path):
    spills = {k: n for k, n in _spills(tmp_path).items() if "k_attn" in k or "k_rope" in k or "k_kv8" in k}
    assert len(spills) >= 26
    assert not {k: n for k, n in spills.items() if n and SPILL not in k}
