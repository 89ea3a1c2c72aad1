"""Norms of wide rows, more of them than workgroups: every workgroup takes further rows,
whose pieces are read ahead and whose sums take turns in LDS."""
import pytest

from test_gpu_norm_residual import Case, env  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("n,dim,dtype", [(600, 4095, "float32"), (513, 2049, "float32"), (1300, 2048, "float32"), (1030, 4096, "bfloat16"),
                                         (700, 2051, "float16"), (2100, 1025, "float32")])
def test_more_rows_than_workgroups(env, kind, n, dim, dtype):  # noqa: F811
    Case(env, n, dim, dtype, kind).check()


def test_wide_rows_of_the_norm_alone_and_without_weights(env):  # noqa: F811
    for kind in ("rms", "layer"):
        Case(env, 600, 4000, "float32", kind, z=False, gate=False, post=False, res=False).check()
        Case(env, 600, 4000, "float32", kind, gate=False, post=False, pre=False).check()
