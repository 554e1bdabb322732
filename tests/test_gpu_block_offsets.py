"""Offsets of a grouped product that break the rules, at sizes where CTAs share a tile's column blocks in clusters and at sizes
where they do not: reported, and every row is written at most once, by the expert that rows_of() (csrc/block_plan.h) gives it."""
import numpy as np
import pytest

from test_gpu_blocks import BF16, E4M3, F32, Matrix, check_product, operands, torch, up16  # noqa: F401 - torch is a fixture
from vpux_plugin_b200 import abi
from vpux_plugin_b200.lib import VfoldError

pytestmark = pytest.mark.gpu


def ranges(offsets, rows):
    reach, out = 0, []
    for a, b in zip(offsets, offsets[1:]):
        lo = max(min(max(a, 0), rows), reach)
        reach = max(min(max(b, 0), rows), lo)
        out.append((lo, reach))
    return out


def garbage(n, seed):
    return [int(v) for v in np.random.default_rng(seed).integers(-2 ** 63, 2 ** 63 - 1, n)]


# rows, offsets, outputs, columns
BAD = [
    (48, [0, 48, 0, 48, 0, 48], 128, 2048),                                         # clusters of eight, one more tile than clusters if rows repeat
    (48, [0, 30, 20, 40, 10, 48], 300, 1153),
    (48, garbage(6, 1), 128, 2048), (48, garbage(41, 2), 128, 2048),
    (128, [0, 128] * 4 + [0], 1024, 4096),                                          # 256 tiles for 128 if rows repeat
    (100, [0, 40, 90, 60, 100], 256, 2048), (100, [0, 60, 0, 101], 200, 1500),      # up to 32 rows per expert, and above
    (300, [0, 250, 100, 301], 128, 4480),
    (70, list(range(0, 33)) + [20] + list(range(33, 69)), 130, 1100),               # a decrease behind the first 32 experts
    (2000, [0, 1500, 700, 2000, 100, 2001], 1100, 512), (2000, [5, 2000] * 20, 300, 300),
]


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("case", range(len(BAD)))
def test_rows_are_owned_once_whatever_the_offsets(gpu, torch, case, aligned):  # noqa: F811
    rows, offsets, n, k = BAD[case]
    rng = np.random.default_rng(100 + case)
    experts = len(offsets) - 1
    ops = operands(rng, rows, n, k, E4M3, E4M3, experts)
    x = Matrix(torch, rows, k, 1, codes=ops[0], scales=ops[1], ld=up16(k), col_major=True)
    w = Matrix(torch, n, k, 128, count=experts, codes=ops[2], scales=ops[3], ld=up16(k) + (0 if aligned else 1))
    out = torch.full((rows, n), 3.0, device="cuda")
    offs = torch.tensor(offsets, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for _ in range(2):
        with pytest.raises(VfoldError) as e:
            gpu.matmul_blocks_grouped(x.pod, w.pod, offs.data_ptr(), out.data_ptr(), F32, out.nbytes)
        assert e.value.status == abi.VF_ERR_RANGE
    got = out.double().cpu().numpy()
    owned = np.zeros(rows, bool)
    for e, (lo, hi) in enumerate(ranges(offsets, rows)):
        check_product(got, *ops, E4M3, E4M3, F32, lo, hi, e)
        owned[lo:hi] = True
    assert (got[~owned] == 3.0).all()


def test_good_offsets_after_bad_ones(gpu, torch):  # noqa: F811
    rng = np.random.default_rng(200)
    ops = operands(rng, 48, 128, 2048, E4M3, E4M3, 5)
    x = Matrix(torch, 48, 2048, 1, codes=ops[0], scales=ops[1], col_major=True)
    w = Matrix(torch, 128, 2048, 128, count=5, codes=ops[2], scales=ops[3])
    out = torch.full((48, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    for offsets, good in (([0, 48, 0, 48, 0, 48], False), ([0, 16, 16, 20, 40, 47], True)):
        out.fill_(3.0)
        offs = torch.tensor(offsets, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        if good:
            gpu.matmul_blocks_grouped(x.pod, w.pod, offs.data_ptr(), out.data_ptr(), BF16, out.nbytes)
        else:
            with pytest.raises(VfoldError):
                gpu.matmul_blocks_grouped(x.pod, w.pod, offs.data_ptr(), out.data_ptr(), BF16, out.nbytes)
    got = out.double().cpu().numpy()
    for e in range(5):
        check_product(got, *ops, E4M3, E4M3, BF16, offsets[e], offsets[e + 1], e)
    assert (got[47:] == 3.0).all()
