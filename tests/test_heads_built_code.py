"""CPU: what the compiler makes of the kernels over ordinary key and value heads and of the page copies, built as the Makefile builds them."""
import pytest

from tests.test_built_code import _built


@pytest.mark.parametrize("source,kernel,count", [("gqa_decode.hip", "gqa_split_kernel", 32), ("heads_prologue.hip", "heads_prologue_kernel", 48),
                                                 ("copy_pages.hip", "copy_pages_kernel", 4)])
def test_no_spills_and_no_flat_accesses(source, kernel, count, tmp_path):
    """Tiles, sums and the next tile's loads fill the registers: what the compiler would put into scratch memory comes back behind a wait
    for every load on its way, and a flat access waits for the LDS as well."""
    bodies = _built(source, kernel, tmp_path)
    assert len(bodies) == count
    for name, body in bodies.items():
        assert not [x for x in body if x.startswith(("scratch_", "flat_load", "flat_store"))], name
