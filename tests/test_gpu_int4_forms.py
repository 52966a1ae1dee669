"""4-bit products at sizes that take each form of the kernels, with every group, ragged in all three sizes, against 64 bits."""
import numpy as np
import pytest

from test_gpu_int4 import Case, check, run

pytestmark = pytest.mark.gpu

# stream forms: 1 x 8, 1 x 16, 2 x 16, 2 x 8, 2 x 4, 2 x 3 tiles x waves
FEW = [(1, 1999, 777), (6, 1999, 4100), (3, 4200, 4097), (8, 4200, 4104), (16, 4200, 4104), (13, 12300, 780), (2, 12301, 1030), (7, 12299, 767)]
# tiles for rows of A at 16 bytes, then for others
MANY = [(33, 1999, 1000), (33, 2999, 1000), (33, 6000, 1000), (33, 700, 264), (33, 700, 136), (257, 3999, 136), (150, 3999, 264), (100, 6001, 4104), (400, 5999, 200)]
ODD = [(17, 99, 6150), (40, 2049, 250), (33, 6000, 130), (33, 6001, 4102), (150, 3999, 4102), (200, 5999, 131)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", FEW + MANY + ODD)
def test_form(pkg, L, m, n, k, group):
    c = Case(m, n, k, group, epi=(m + group // 32) % 3)
    got = check(pkg, L, c)
    if c.epi == 2:
        np.testing.assert_array_equal(run(pkg, L, c, in_place=True), got)
