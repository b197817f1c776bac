"""CPU: what the compiler makes of the kernels of a step over drafted trees, built as the Makefile builds them."""
import pytest

from tests.test_built_code import _built


@pytest.mark.parametrize("source,kernel,count", [("gqa_tree.hip", "gqa_split_kernel", 32), ("gqa_wide.hip", "gqa_tree_wide_kernel", 12),
                                                 ("keep_rows.hip", "keep_rows_kernel", 4), ("step_tables.hip", "kernel", 2)])
def test_no_spills_and_no_flat_accesses(source, kernel, count, tmp_path):
    """Tiles, sums and loads under way fill the registers: what the compiler would put into scratch memory comes back behind a wait for every load on its
    way, and a flat access waits for the LDS as well."""
    bodies = _built(source, kernel, tmp_path)
    assert len(bodies) == count
    for name, body in bodies.items():
        assert not [x for x in body if x.startswith(("scratch_", "flat_load", "flat_store"))], name
