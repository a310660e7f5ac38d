"""8-bit integer products through every kernel that their size chooses, and the command that generates text."""
import pytest
import torch

from helpers import announce
from test_generate_ops_gpu import check_linear, operands

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]

# few_kernel: tokens quantised by one, two and half a wave each, read quantised for 16 and 32 rows; rows quantised by a
# wave that holds 4096; 64-tiles; 128-tiles alone; 128- and 256-tiles, their outputs below and above 32 MB; n of no 8
PRODUCTS = [(1, 2048, 512), (7, 4001, 130), (8, 4096, 1024), (8, 1024, 512), (16, 700, 90), (31, 1000, 90),
            (12, 3000, 100), (31, 2000, 100), (32, 4500, 72), (2100, 1500, 40), (2049, 4096, 24),
            (100, 1001, 300), (65, 1024, 32001), (65, 700, 32000), (2100, 1024, 3081), (2100, 300, 3088),
            (2049, 128, 3968), (2049, 128, 3967), (4096, 128, 4096), (8000, 256, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_every_product_kernel(dtype, m, k, n):
    announce(f"product {dtype} {m} {k} {n}")
    x, w, b, r = operands(m, k, n, dtype)
    check_linear(x, w, b, r, gelu=True)
    if m * n < 1 << 20:
        check_linear(x, w)
        check_linear(x, w, b, None, ldx=k + 3, offset=1)
        check_linear(x, w, None, r, ldr=n + 5, offset=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,n", [(2048, 4000), (640, 4001)])
def test_rows_alone_and_among_others(dtype, k, n):
    """A row's bits are the same from every kernel."""
    from ceo_amd import nn

    announce(f"rows {dtype} {k} {n}")
    x, w, b, r = (t.cuda() for t in operands(2100, k, n, dtype))
    wt = nn.Int8Weight(w)
    for gelu in (False, True):
        full = nn.linear_int8(x, wt, b, r, gelu)
        for m in (1, 8, 9, 16, 17, 32, 33, 64, 200, 1000, 1100):
            assert torch.equal(nn.linear_int8(x[:m], wt, b, r[:m], gelu), full[:m]), m


@pytest.mark.parametrize("m", [3, 40, 100])
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_of_the_largest_values(dtype, m):
    x, w, b, r = operands(m, 300, 40, dtype)
    x[2] = torch.finfo(dtype).max / 4
    x[1, 7] = torch.finfo(dtype).max
    w = (w.float() * (1e-3 if dtype is torch.float16 else 1e-38)).to(dtype)
    check_linear(x, w)
    check_linear(x, w, b, r, gelu=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(3, 500, 72), (8, 4096, 64), (31, 2000, 100), (100, 1001, 304), (65, 300, 32000),
                                   (2100, 300, 3088), (2049, 128, 3968), (2049, 128, 3967), (4096, 128, 4096)])
def test_output_over_its_residual(dtype, m, k, n):
    from ceo_amd import _lib, nn

    announce(f"residual in place {dtype} {m} {k} {n}")
    x, w, b, r = (t.cuda() for t in operands(m, k, n, dtype))
    wt = nn.Int8Weight(w)
    want = nn.linear_int8(x, wt, b, r)
    code = {torch.bfloat16: 14, torch.float16: 2, torch.float32: 0}[dtype]
    assert _lib.lib().linear_int8_hip(x.data_ptr(), k, wt.packed.data_ptr(), b.data_ptr(), r.data_ptr(), n, r.data_ptr(),
                                      n, m, k, n, 0, code, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(r, want)


def test_the_command_runs(capsys):
    from ceo_amd import generate

    generate.main()
    lines = capsys.readouterr().out.splitlines()
    assert lines[0].startswith("counting: loss")
    assert [x for x in lines if x.endswith(":")] == ["bf16 products:", "8-bit products:"]
    texts = [x for x in lines if "|" in x]
    assert len(texts) == 4
    for x in texts:
        prompt, rest = x.split("|")
        new, score = rest.split("(")
        assert prompt.split() in (["7", "8", "9", "10"], ["200", "201", "202", "203"])
        assert len(new.split()) == 12 and all(0 <= int(v) < 256 for v in new.split())
        assert float(score.rstrip(")")) <= 0.0
