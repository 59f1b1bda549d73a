"""What gsp_matmul_batch_fp8 keeps of device memory."""
import pytest

from fp8_helpers import Q4_1

pytestmark = pytest.mark.gpu


def test_converted_activations_do_not_double_past_a_gigabyte(torch_mod, gsp):
    """A product of 0.93 GB, then one of the most, 1.07 GB: the context keeps 1.07 GB and the split sums' few MB."""
    torch = torch_mod
    ctx = gsp.Context(0)
    in_dim, out_dim = 131072, 520
    w = torch.zeros((out_dim, in_dim // 32 * 20), dtype=torch.uint8, device="cuda")
    x = torch.zeros((9001, in_dim), dtype=torch.uint8, device="cuda")
    s, y = torch.ones(9001, device="cuda"), torch.ones((9001, out_dim), device="cuda")
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    kept = []
    for batch in (3300, 9001):
        ctx.matmul_batch_fp8(Q4_1, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
        ctx.sync()
        kept.append(free - torch.cuda.mem_get_info()[0])
    print(f"kept {kept}", flush=True)
    assert not y.any()
    assert 0.9e9 < kept[0] <= 1.0e9 and 1.0e9 < kept[1] <= 1.15e9
    ctx.close()
    del x, w
    torch.cuda.empty_cache()
