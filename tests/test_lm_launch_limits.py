"""Sizes whose launches have more threads than a launch counts (32 bits along a
dimension of the grid) are refused before the first of an operator's kernels.
Called with made-up addresses, so without a GPU only: the largest size that is
let pass ends at the missing device."""
import pytest

from neon_amd.backends.hip import runtime as hiprt

pytestmark = pytest.mark.skipif(hiprt.device_count() > 0, reason="a device is there: the good calls would run on made-up addresses")

P, BIG = 4096, 1 << 60
F32, F16 = 0, 1
B256, B512, B1024 = ((1 << 32) // t - 1 for t in (256, 512, 1024))       # workgroups a launch counts


def ln_fprop(lib, dtype, axis, f, n):
    ld = f if axis else n
    return lib.nh_ln_fprop(P, P, P, P, P, P, 1e-5, dtype, axis, f, n, ld, ld, P, BIG, None)


def ln_bprop(lib, dtype, axis, f, n):
    ld = f if axis else n
    return lib.nh_ln_bprop(P, P, P, P, P, P, P, P, 1e-5, dtype, axis, f, n, ld, ld, ld, P, BIG, None)


def embed_fprop(lib, dtype, axis, e, n):
    return lib.nh_embed_fprop(P, P, P, 1.0, dtype, axis, n, e, 1000, e, e if axis else n, -1, None)


def embed_update(lib, dtype, axis, e, n, vocab=1000, beta=0.0):
    return lib.nh_embed_update(P, P, P, 1.0, beta, dtype, axis, n, e, vocab, e, e if axis else n, -1, P, BIG, None)


def clear(lib, dtype, axis, e, vocab):
    return embed_update(lib, dtype, axis, e, 50, vocab)


def distill_fprop(lib, dtype, axis, v, n):
    s = hiprt.int64s(1, 1, 1, 1, 1, 1, 1)
    return lib.nh_distill_fprop(P, P, P, P, P, 1.0, dtype, dtype, axis, v, n, 3, v if axis else n, s, P, BIG, None)


def distill_bprop(lib, dtype, axis, v, n, k=3):
    s, ld = hiprt.int64s(1, 1, 1, 1, 1, 1, 1), v if axis else n
    return lib.nh_distill_bprop(P, P, P, P, P, None, 1.0, 1.0, dtype, dtype, axis, v, n, k, ld, ld, s, None)


def without_entries(lib, dtype, axis, v, n):
    return distill_bprop(lib, dtype, axis, v, n, 0)


@pytest.mark.parametrize("call,dtype,axis,width,most", [
    (ln_fprop, F32, 1, 40000, B1024), (ln_fprop, F16, 1, 20000, B1024),           # a workgroup per row
    (ln_fprop, F16, 0, 100, 64 * B256), (ln_fprop, F16, 0, 1000, 32 * B512), (ln_fprop, F16, 0, 2000, 32 * B1024),
    (ln_fprop, F32, 0, 3000, 32 * B256),
    (ln_bprop, F32, 1, 9000, B1024), (ln_bprop, F16, 0, 100, 32 * B256), (ln_bprop, F32, 0, 2000, 16 * B1024),
    (embed_fprop, F16, 1, 2048, B256), (embed_fprop, F16, 0, 64, 128 * B256),
    (clear, F32, 1, 1, 64 * (B256 - 3)),              # (three workgroups look for words and add)
    (distill_fprop, F32, 1, 10, B256), (distill_fprop, F32, 0, 10, 16 * B256),
    (distill_bprop, F32, 1, 10, B256), (distill_bprop, F32, 0, 10, 8 * B256), (without_entries, F32, 0, 10, 64 * B256)])
def test_the_largest_launch(call, dtype, axis, width, most):
    lib = hiprt.load_library()
    assert call(lib, dtype, axis, width, most) == hiprt.NH_ENOTINIT
    assert call(lib, dtype, axis, width, most + 1) == hiprt.NH_EINVAL
    assert b"threads" in lib.nh_last_error()


def test_more_features_than_the_parameter_sums_launch():
    lib = hiprt.load_library()
    for axis in (0, 1):
        assert ln_bprop(lib, F16, axis, 32 * B1024, 2) == hiprt.NH_ENOTINIT
        assert ln_bprop(lib, F16, axis, 32 * B1024 + 1, 2) == hiprt.NH_EINVAL


def test_errors_turned_around_by_more_workgroups_than_a_launch_has():
    """64 GiB of errors in the columns layout: nothing may run on the table of
    classes that the refused launch would have written"""
    lib = hiprt.load_library()
    assert embed_update(lib, F16, 0, 1024, 33000000) == hiprt.NH_ENOTINIT
    assert embed_update(lib, F16, 0, 1024, 1 << 25) == hiprt.NH_EINVAL
    assert embed_update(lib, F16, 1, 1024, 1 << 25) == hiprt.NH_ENOTINIT          # nothing to turn in rows
    # beta = 1 leaves absent words alone, whatever their number
    assert embed_update(lib, F32, 1, 1, 50, 0x7FFFFFFF, 1.0) == hiprt.NH_ENOTINIT


def test_walking_workgroups_have_no_such_limit():
    lib = hiprt.load_library()
    for call in (ln_fprop, ln_bprop):
        assert call(lib, F16, 1, 1000, 1 << 40) == hiprt.NH_ENOTINIT
