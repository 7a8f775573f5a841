"""The limits of the grouped products that are a matter of sizes alone, asked for without a device: a call with sizes inside them gets
as far as a later refusal."""
import pytest


@pytest.fixture(scope="module")
def L():
    from unit_amd import _lib
    return _lib.load()


# N x K below, between and above 2^29 and 2^30 elements: 2^31 bytes in fp32 and in 16 bits
@pytest.mark.parametrize("n,k,inside", [(8192, 8192, True), (16392, 32776, True), (248, 1 << 22, True), (32768, 32760, True), (32768, 32768, False)])
@pytest.mark.parametrize("out_dtype", [0, 1])
def test_a_weight_has_a_gradient_where_it_has_a_product(L, n, k, inside, out_dtype):
    for f in (L.unit_grouped_dense, L.unit_grouped_dense_grad_data, L.unit_grouped_dense_grad_weight):
        rc = f(16, 16, 16, 4, 8, 1, out_dtype, 4, 2, n, k, None)  # a result off 16 bytes
        said = L.unit_last_error().decode()
        assert rc == -1 and ("aligned" in said if inside else "2^31" in said), (f, said)
