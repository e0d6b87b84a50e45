"""What the Python package needs and takes: dtypes of torch tensors."""
import pytest
import torch


@pytest.fixture(scope="module")
def F(built_libs):
    from diopi_b200 import functions
    return functions


def test_float8_tensors_only_where_codes_are_meant(F):
    """The interface has no 8-bit float. An op without e4m3 codes does not take them for whole numbers."""
    x = torch.zeros(3, 2, 8).to(torch.float8_e4m3fn)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        F.destindex_copy_kv(x, torch.zeros(3, dtype=torch.int32), x.clone(), as_device=True)
    from diopi_b200.runtime import Tensor
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        Tensor(x, as_device=True)
    # the caches of the 8-bit operators are: what is refused here is the next argument
    from diopi_b200.runtime import DiopiError
    cache, scale, ids = torch.zeros(4, 16, 2, 8).to(torch.float8_e4m3fn), torch.zeros(4, 2), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(DiopiError, match="softmax_scale"):
        F.quantized_paged_attention(torch.zeros(1, 2, 8).half(), cache, cache, scale, scale, ids, ids[0, :1], -1.0, as_device=True)
