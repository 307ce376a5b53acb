"""Soft code assignment, balance loss and distillation where their arithmetic can go wrong: sums that are whole numbers and have to
come out exactly, sums that cancel, infinities and the largest values, empty batches, high temperatures.  Bounds as in
tests/loss_utils.py: U = 2^-24, half a step of the result's type where it is stored."""
import importlib
import math

import pytest
import torch

from loss_utils import U, assert_within, store_error

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def eng():
    return importlib.import_module("gan-discovery-pso_amd.engine")


@pytest.fixture(scope="module")
def fn():
    return importlib.import_module("gan-discovery-pso_amd.inverter.utils_vq_vae.util_function")


def generator(seed):
    return torch.Generator().manual_seed(seed)


def rand(seed, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=generator(seed)) * scale).to(dtype).to(DEV)


def whole(seed, most, *shape, dtype=torch.float32):
    """Whole numbers in [-most, most]."""
    return torch.randint(-most, most + 1, shape, generator=generator(seed)).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------------------- code gradients
def three_entries(seed, rows, cols):
    """[rows, cols] with three entries a row that sum to nothing, up to their own rounding."""
    gen = generator(seed)
    at = torch.stack([torch.randperm(cols, generator=gen)[:3] for _ in range(rows)])
    v = torch.randn(rows, 2, generator=gen)
    v = torch.cat([v, -v.sum(dim=1, keepdim=True)], dim=1)
    return torch.zeros(rows, cols).scatter_(1, at, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,d", [(40, 30, 20), (5000, 300, 64), (4500, 1000, 130), (33000, 130, 24)])
def test_code_gradients_of_sums_that_cancel(eng, n, k, d, dtype):
    """Rows (columns) of three entries that sum to nothing, times codes (latents) of one large offset: what is left is 2^-10 of the
    summands for fp16.  A sum of three whole products meets three roundings of at most one step, 2 U, of the summands' magnitudes, and
    the result two more of its own, so it is off by at most 8 U of the magnitudes; a logits' gradient held in fewer bits than
    its own 24 would not cancel (16 bits: 64 U)."""
    offset = {torch.float32: 2.0 ** 20, torch.bfloat16: 128.0, torch.float16: 1024.0}[dtype]
    code = (offset + whole(1, 3, k, d).abs()).to(dtype)
    x = (offset + whole(2, 3, n, d).abs()).to(dtype)
    c64, x64 = code.double().cpu(), x.double().cpu()
    g = three_entries(3, n, k)
    dx, _ = eng.code_logits_grad(g.to(DEV), x, code, temperature=2.0, want_codebook=False)
    g = g.double()
    want = g @ c64
    assert_within(dx, want, (g.abs() @ c64.abs()) * 8 * U + store_error(want, dtype), "dx")
    g = three_entries(4, k, n).t().contiguous()
    _, dc = eng.code_logits_grad(g.to(DEV), x, code, temperature=2.0, want_inputs=False)
    g = g.double()
    want = g.t() @ x64 - g.sum(dim=0)[:, None] * c64
    assert_within(dc, want, (g.abs().t() @ x64.abs()) * 8 * U + (g.sum(dim=0).abs() + 3 * U * g.abs().sum(dim=0))[:, None] * c64 * 2 * U
                  + g.abs().sum(dim=0)[:, None] * c64 * 3 * U + store_error(want, dtype), "dcode")


# Every form of the three products: sizes around the rules that choose tiles, splits and stages, with cut last tiles and sums.
WHOLE_SIZES = [(1, 1, 1), (33, 31, 17), (512, 256, 100), (2049, 130, 65), (4097, 257, 33), (5000, 40, 300), (8193, 129, 64), (9001, 300, 150),
               (9002, 515, 180), (8195, 1025, 210), (8200, 700, 250), (8199, 333, 256), (9000, 260, 300), (9000, 1500, 256), (20001, 64, 31),
               (32769, 65, 20), (32775, 512, 64), (33001, 513, 128), (50007, 1024, 48), (66001, 33, 130), (100003, 1000, 10)]


def check_whole(eng, n, k, d, dtype):
    x, code, g = whole(n, 3, n, d, dtype=dtype), whole(k, 3, k, d, dtype=dtype), whole(d, 3, n, k)
    x64, c64, g64 = x.double().cpu(), code.double().cpu(), g.double().cpu()
    assert torch.equal(eng.code_logits(x, code, temperature=2.0).double().cpu(), x64 @ c64.t() - (c64 * c64).sum(dim=1) / 2)
    dx, dc = eng.code_logits_grad(g, x, code, temperature=2.0)
    assert torch.equal(dx.cpu(), (g64 @ c64).to(dtype))
    assert torch.equal(dc.cpu(), (g64.t() @ x64 - g64.sum(dim=0)[:, None] * c64).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,d", WHOLE_SIZES)
def test_code_products_of_whole_numbers_are_exact(eng, n, k, d, dtype):
    """All partial sums are whole numbers (or halves) below 2^24, which fp32 holds: a lost row, stage, split or part shows."""
    check_whole(eng, n, k, d, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_code_gradients_of_whole_numbers_are_exact(eng, dtype):
    check_whole(eng, 16411, 4099, 256, dtype)  # above 2^34 products


@pytest.mark.parametrize("n,k,d", [(70, 40, 24), (300, 64, 200), (5000, 130, 40), (9001, 70, 150), (33000, 64, 64)])
def test_code_products_with_infinities_and_the_largest_values(eng, n, k, d):
    """fp32 values that a 16-bit type rounds up to infinity stay finite, and an infinity reaches what the formula says."""
    biggest = torch.finfo(torch.float32).max
    x, code = rand(n, n, d), rand(k, k, d, scale=1e-3)
    g = rand(d, n, k)
    x[3, 5], x[4, 2] = math.inf, -math.inf
    x[6], x[7, 1] = -biggest, biggest  # padding rows of the type's lowest value, with a gradient of 0
    code[2, 7] = 0.0
    code[11, 9] = math.inf
    g[6:8] = 0.0
    g[9, 4], g[10, 4] = math.inf, biggest * 1e-2
    s = eng.code_logits(x, code).double().cpu()
    x64, c64, g64 = x.double().cpu(), code.double().cpu(), g.double().cpu()
    want = 2 * x64 @ c64.t() - (c64 * c64).sum(dim=1)
    bound = (2 * x64.abs() @ c64.abs().t() + (c64 * c64).sum(dim=1)) * (d + 4) * U + store_error(want, torch.float32)
    big = want.abs() > 2 * biggest
    want[big] = want[big].sign() * math.inf

    def check(got, want, bound, what):
        finite = want.isfinite()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~finite].nan_to_num(nan=7.0), want[~finite].nan_to_num(nan=7.0)), what
        assert_within(got[finite], want[finite], bound[finite], what)

    check(s, want, bound, "logits")
    dx, dc = (t.double().cpu() for t in eng.code_logits_grad(g, x, code))
    want = 2 * g64 @ c64
    check(dx, want, 2 * (g64.abs() @ c64.abs()) * (k + 4) * U + store_error(want, torch.float32), "dx")
    want = 2 * (g64.t() @ x64 - g64.sum(dim=0)[:, None] * c64)
    bound = 2 * (g64.abs().t() @ x64.abs() + g64.abs().sum(dim=0)[:, None] * c64.abs()) * (n + 8) * U + store_error(want, torch.float32)
    check(dc, want, bound, "dcode")


# -------------------------------------------------------------------------------------------------- empty batches
@pytest.mark.parametrize("v", [8, 3000, 20000, 200003])
@pytest.mark.parametrize("masked", [False, True])
def test_distill_of_no_rows(v, masked):
    """Loss and stats are written whatever the buffers held before."""
    lib = importlib.import_module("gan-discovery-pso_amd._lib")
    L = lib.lib()
    size = L.gdpso_distill_workspace_bytes(0, v, 4)
    ws = torch.full((size // 4 + 4,), math.nan, device=DEV)
    loss, stats = torch.full((), math.nan, device=DEV), torch.full((1,), math.nan, device=DEV)
    mask = torch.ones(1, dtype=torch.uint8, device=DEV) if masked else None
    lib.run(loss.device, L.gdpso_distill, 0, v, 4, None, v, 0, None, 0, None, 8, lib.ptr(mask), 1.0, 1.0, loss.data_ptr(), None, stats.data_ptr(), None,
            ws.data_ptr(), size)
    assert float(loss) == 0.0 and float(stats) == 0.0
