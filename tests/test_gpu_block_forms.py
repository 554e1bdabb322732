"""Every form of the products (csrc/block_plan.h) against the definition where it works longest: several tiles per CTA, more column
blocks than the rings of scales and stages hold, last tiles with few rows and columns, every type, result pitches that do and do not
allow 16-byte stores. A size that no longer reaches the form it is named for fails."""
import numpy as np
import pytest

import block_reference as br
from test_block_plan_cpu import forms_of
from test_gpu_blocks import BF16, E4M3, E5M2, F16, F32, check_product, run_product, torch  # noqa: F401 - torch is a fixture

pytestmark = pytest.mark.gpu

TYPES = [(E4M3, E4M3, BF16), (E5M2, E4M3, F16), (E4M3, E5M2, F32)]



def made(torch, seed, m, n, k, xt, wt, count=1):  # noqa: F811
    """Codes of bell-shaped values (torch's conversion) and scales over a factor of four: quantising as many in 64 bits takes long."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def codes(shape, dtype):
        t, sigma = (torch.float8_e4m3fn, 100.0) if dtype == E4M3 else (torch.float8_e5m2, 1e4)
        v = (torch.randn(shape, generator=g, device="cuda") * sigma).clamp(-br.LARGEST[dtype], br.LARGEST[dtype])
        return v.to(t).view(torch.uint8).cpu().numpy()

    def scales(shape, dtype, size):
        return (torch.exp2(torch.rand(shape, generator=g, device="cuda") * 2 - 1) * (size / (100.0 if dtype == E4M3 else 1e4))).cpu().numpy()

    kb = -(-k // 128)
    return codes((m, k), xt), scales((m, kb), xt, 1.0), codes((count, n, k), wt), scales((count, -(-n // 128), kb), wt, 0.02)


# form, rows, outputs, columns, pitch of the result beyond the outputs
DENSE = [
    ("Wide256", 3001, 2900, 1300, 0), ("Wide256", 3001, 2900, 2700, 1), ("Wide256", 2500, 3000, 1100, 8),  # 276, 240 tiles; last ones of 84, 184 columns
    ("Wide256", 2433, 3201, 2200, 0),                                                                     # a last tile of one row and 129 columns
    ("Wide128", 1500, 4096, 1300, 0), ("Wide128", 1537, 3900, 2700, 3), ("Wide128", 700, 1501, 2300, 8),
    ("Swap128", 300, 1000, 2700, 1), ("Swap128", 500, 1024, 4480, 0),
    ("Swap32", 40, 3000, 4480, 0), ("Swap32", 29, 20000, 1300, 3), ("Swap16", 9, 30001, 2700, 0),
]


@pytest.mark.parametrize("types", range(len(TYPES)))
@pytest.mark.parametrize("case", range(len(DENSE)))
def test_form(gpu, torch, case, types):  # noqa: F811
    form, m, n, k, more = DENSE[case]
    xt, wt, out_dt = TYPES[types]
    assert forms_of([(m, 0, n, torch.cuda.get_device_properties(0).multi_processor_count)]) == [form]
    ops = made(torch, 300 + case, m, n, k, xt, wt)
    got = run_product(gpu, torch, *ops, xt, wt, out_dt, out_ld=n + more if more else 0, out_offset=more % 8)
    check_product(got, *ops, xt, wt, out_dt)


def spread(total, experts, seed):
    """Offsets of experts that are chosen unevenly; some get no row, and a few rows belong to nobody."""
    rng = np.random.default_rng(seed)
    p = 1.0 / (np.arange(experts) + 1.0)
    p[1] = 0
    counts = rng.multinomial(total, p / p.sum())
    return [3] + [int(v) + 3 for v in counts.cumsum()]


GROUPED = [
    ("Wide256", 3000, 5, 2900, 1300, 0), ("Wide256", 2600, 7, 3001, 2200, 1), ("Wide256", 2048, 40, 2100, 1100, 8),
    ("Wide128", 901, 7, 1410, 2300, 0), ("Wide256", 1400, 6, 1501, 1300, 3), ("Wide128", 1000, 5, 1501, 1300, 3),
    ("Swap128", 330, 4, 700, 2700, 1), ("Swap32", 150, 5, 1000, 4480, 0), ("Swap16", 70, 9, 1400, 2700, 3), ("Swap16", 40, 64, 1024, 2048, 0),
]


@pytest.mark.parametrize("types", range(len(TYPES)))
@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_grouped_form(gpu, torch, case, types):  # noqa: F811
    form, total, experts, n, k, more = GROUPED[case]
    xt, wt, out_dt = TYPES[types]
    offsets = spread(total, experts, case)
    m = offsets[-1] + 5
    assert forms_of([(m, experts, n, torch.cuda.get_device_properties(0).multi_processor_count)]) == [form]
    ops = made(torch, 400 + case, m, n, k, xt, wt, experts)
    got = run_product(gpu, torch, *ops, xt, wt, out_dt, offsets=offsets, out_ld=n + more if more else 0, out_offset=more % 8)
    for e in range(experts):
        check_product(got, *ops, xt, wt, out_dt, offsets[e], offsets[e + 1], e)
    assert (got[:3] == 3).all() and (got[-5:] == 3).all()
