"""The host side of include/pmg_lm.h at the ends of what it allows, on a machine without a GPU: no compute call is made."""
import ctypes as C

FAKE = 1 << 20          # an aligned address that nothing reads


def test_empty_tensors_overlap_nothing():
    """Tensors cut from one flat buffer: an empty one may point at the start of another, into it, or behind it."""
    from paccmann_generator_amd import _ffi
    check = _ffi.lib.pmg_grad_clip_check

    def rc(ptrs, numel):
        n = len(ptrs)
        return check((C.c_void_p * n)(*ptrs), (C.c_int64 * n)(*numel), (C.c_int * n)(*([0] * n)), n, 1.0)

    for at in (0, 4, 8, 128, 252, 256):
        assert rc([FAKE, FAKE + at], [64, 0]) == 0 and rc([FAKE + at, FAKE], [0, 64]) == 0, at
        # two hundred of them at one place, among tensors that touch
        many = [FAKE + at] * 200
        assert rc(many + [FAKE, FAKE + 256], [0] * 200 + [64, 8]) == 0, at
        assert rc([FAKE, FAKE + 256] + many, [64, 8] + [0] * 200) == 0, at
        bad = rc(many + [FAKE, FAKE + 252], [0] * 200 + [64, 8])
        assert bad < 0 and b'overlap' in _ffi.lib.pmg_strerror(bad)
    assert rc([FAKE, FAKE], [0, 0]) == 0 and rc([None, FAKE], [0, 4]) == 0
