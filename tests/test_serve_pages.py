"""The serving loop's pages, without a GPU."""
import pytest

import fmha_native_b200 as fm


def test_a_refused_extension_changes_nothing():
    from fmha_native_b200.serve import PagedKV

    for slots, max_pages, new in ((2, 8, [16, 80]), (2, 2, [16, 33]), (3, 3, [40, 16, 16])):
        kv = PagedKV(1, 4, 16, 2, slots, max_pages, "cpu")
        kv.extend([1] + [0] * (slots - 1))
        before = (list(kv.free), [list(x) for x in kv.owned], list(kv.host_lengths), kv.host_table.clone())
        with pytest.raises(fm.FmhaError):
            kv.extend(new)
        assert (kv.free, kv.owned, kv.host_lengths) == before[:3] and (kv.host_table == before[3]).all()
        kv.extend([15] + [0] * (slots - 1))
        assert kv.lengths.tolist() == [16] + [0] * (slots - 1) and len(kv.owned[0]) == 1
        kv.extend([1] + [0] * (slots - 1))
        assert len(kv.owned[0]) == 2 and kv.table[0, :2].tolist() == kv.owned[0]
        kv.release(0)
        assert len(kv.free) == 4
