"""The matrix instructions that the tall blocks' products in 8-bit integers write out themselves (csrc/gemm_q8_tall.hip), looked at as those in
bfloat16 are."""
from tests import test_rows_tall_listing


def test_no_vector_instruction_beside_a_product_of_integers(tmp_path):
    test_rows_tall_listing.test_no_vector_instruction_beside_a_product("gemm_q8_tall", 15, tmp_path)
