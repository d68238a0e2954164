"""The layer operators of include/nemo_ops.h at the ends of their ranges."""
import pytest
import torch

import layer_ops_ref as ref
from layer_ops_ref import F32

pytestmark = pytest.mark.gpu


@pytest.fixture
def gen():
    g = torch.Generator(device="cuda")
    g.manual_seed(78)
    return g


# --- w4_matvec -------------------------------------------------------------------

@pytest.mark.parametrize("m,n", [(1, 50000), (2, 50000), (3, 500)])
@pytest.mark.parametrize("shift", [-96, -110, -122])
def test_w4_matvec_of_the_smallest_bf16_values(gen, shift, m, n):
    """Rows whose largest element is near 2^shift, down to subnormal ones. As check_w4, but without an absolute term
    other than that of subnormal f32 sums: 2^-150 for each of at most 4 products a segment and 64 more additions."""
    k, group = 1024, 128
    x = torch.randn((m, k), generator=gen, device="cuda", dtype=torch.float64)
    x = (x * 2.0 ** (shift + torch.randint(-10, 1, (m, k), generator=gen, device="cuda"))).bfloat16()
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
    z = torch.randint(0, 16, (n, k // group), generator=gen, device="cuda")
    s = (4 * torch.randn((n, k // group), generator=gen, device="cuda")).half()
    y = ref.w4_matvec(x, None, 0, ref.pack4(q), s, ref.pack4(z), group, n, F32)
    w = (q.double() - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)
    want, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    segments = k // group
    slack = (40 + segments / 4) * 2 * ref.U32 * mag + (64 + 4 * segments) * 2.0 ** -150
    ref.close(y, want, ref.U32 * want.abs() + slack)
