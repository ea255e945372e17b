"""Token counts on the GPU that hold more rows than there are, up to sums beyond 32 bits: the products
cut them where the rows end, compute the rows of the segments before that, touch nothing else and report
the mismatch."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS, EXPERTS, N, K = 2_200_000, 1024, 8, 16  # 1024 times the rows: past 2^31


def small_integers(shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-3, 4, shape, device=DEV, generator=g)


@pytest.fixture(scope="module")
def operands():
    x, w = small_integers((ROWS, K), 0), small_integers((EXPERTS, N, K), 1)
    return x, w, (x.float() @ w[0].float().t()).to(torch.bfloat16)  # |sum| <= 144: exact in bf16


def wild_counts():
    c = torch.full((EXPERTS,), ROWS, device=DEV)
    big = c.clone()
    big[1:] = 1 << 62
    return [c, big]


@pytest.mark.parametrize("tc", [4, 0, 1, 3])
@pytest.mark.parametrize("int8", [False, True])
def test_sums_past_32_bits(operands, tc, int8):
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt, grouped_gemm_opt_int8
    x, w, want = operands
    check_device_errors(0)
    for counts in wild_counts():
        for sort in (True, False):
            if int8:
                out = grouped_gemm_opt_int8(x.to(torch.int8), torch.ones(ROWS, device=DEV),
                                            w.to(torch.int8), torch.ones(EXPERTS, N, device=DEV),
                                            counts, tc, sort)
            else:
                out = grouped_gemm_opt(x.to(torch.bfloat16), w.to(torch.bfloat16), counts, tc, sort)
            assert torch.equal(out, want)
            with pytest.raises(RuntimeError):
                check_device_errors(0)
    check_device_errors(0)


@pytest.mark.parametrize("tc", [4, 0, 1, 3])
def test_a_segment_is_cut_where_the_rows_end(tc):
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt
    counts = [300, 20, 500, 40]  # 700 rows
    x = small_integers((700, 64), 2).to(torch.bfloat16)
    w = small_integers((4, 256, 64), 3).to(torch.bfloat16)
    out = grouped_gemm_opt(x, w, torch.tensor(counts, device=DEV), tc)
    with pytest.raises(RuntimeError):
        check_device_errors(0)
    at = 0
    for e, c in enumerate([300, 20, 380]):
        want = (x[at:at + c].float() @ w[e].float().t()).to(torch.bfloat16)
        assert torch.equal(out[at:at + c], want)
        at += c


def test_block_scales_past_32_bits():
    """Only the first segment has rows; scales and codes are those of counts that say so."""
    from grouped_gemm_opt import quantize_mxfp8
    x = small_integers((ROWS, 128), 4).to(torch.bfloat16)
    right = torch.zeros(EXPERTS, dtype=torch.int64, device=DEV)
    right[0] = ROWS
    q, s = quantize_mxfp8(x, right)
    for counts in wild_counts():
        got_q, got_s = quantize_mxfp8(x, counts)
        assert torch.equal(got_q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(got_s, s)
