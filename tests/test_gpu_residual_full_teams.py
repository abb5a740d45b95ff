"""Residual blocks of 4097 to 8192 values, whose forward holds its parameters packed in LDS: teams with all lanes in use and with
a partial last chunk, and either side of the room that five, four and fewer parameters take (up to 8152 values with five)."""
import pytest

from test_gpu_residual import ALL, BF16, F32, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dim", [4097, 6000, 7001, 8145, 8152, 8153, 8160, 8185, 8191, 8192])
def test_all_parts(dim, norm):
    check(5, dim, F32, F32, F32, ALL, norm)
    check(3, dim, BF16, BF16, BF16, ALL, norm, drop=0.3, seed=2)
    check(3, dim, F32, BF16, F32, ALL, norm, seed=3)


@pytest.mark.parametrize("parts", [{"next"}, {"next", "bias"}, {"y", "post", "next", "rows"}, {"y", "post", "next", "bias", "rows"},
                                   {"y", "post", "next", "gate"}, {"y", "rows"}], ids=lambda p: "-".join(sorted(p)))
@pytest.mark.parametrize("dim", [4100, 6001, 8153, 8185, 8192])
def test_fewer_parts(parts, dim):
    check(4, dim, F32, F32, F32, parts, "layer", drop=0.2 if "y" in parts else 0.0)
    check(4, dim, BF16, BF16, F32, parts, "rms", seed=2)
    check(300, dim, BF16, F32, BF16, parts, "layer", seed=3)
