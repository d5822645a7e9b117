"""The first size that each entry point of the mixers refuses because its launch would have 2^32
threads, and the last one before it: that one gets as far as the check of its (null) tensors."""
import pytest

from hattention import _lib

VAL, NOT = _lib.HATTN_ERR_VALUE, _lib.HATTN_ERR_NOT_IMPLEMENTED
BF, FS = 0, 2
MAX = 2 ** 31 - 1


def code(name, *args):
    return getattr(_lib.load(), name)(*args)


# B, T, D, dtype and whether the scan is refused: rows x segments x strips of 64 channels, or 128
@pytest.mark.parametrize("B,T,D,dtype,refused", [
    (2 ** 23, 1, 1, FS, True), (2 ** 23 - 1, 1, 1, FS, False), (2 ** 23 - 1, 256, 64, FS, False),
    (2 ** 22, 257, 64, FS, True), (2 ** 22 - 1, 257, 64, FS, False), (2 ** 22, 1, 65, FS, True),
    (2 ** 22, 1, 66, BF, False), (2 ** 23, 1, 66, BF, True), (2 ** 22, 129, 66, BF, True),
    (2 ** 22, 129, 65, BF, True), (2 ** 22, 128, 65, BF, True), (2 ** 22, 256, 63, BF, False),
    (1, 1, MAX, FS, True), (1, 2 ** 30, 1, FS, False), (2, 2 ** 30, 1, FS, True),
    (MAX, 1, MAX, FS, True)])
def test_recurrence(B, T, D, dtype, refused):
    want = NOT if refused else VAL
    assert code("hattn_gated_recurrence_fwd", *([None] * 7), B, T, D, dtype, dtype, None, 0, None) == want
    assert code("hattn_gated_recurrence_bwd", *([None] * 9), B, T, D, dtype, dtype, None, 0, None) == want
    segments = _lib.load().hattn_gated_recurrence_segments(T, D, dtype)
    assert segments == 0 if refused and B == 1 else segments > 0 or D == MAX
    assert _lib.load().hattn_gated_recurrence_workspace(B, T, D, dtype) == 0 or not refused


@pytest.mark.parametrize("B,D,refused", [
    (2 ** 16, 2 ** 16, True), (2 ** 16, 2 ** 16 - 1, False), (2, MAX, True), (1, MAX, False),
    (2 ** 23, 1, False), (MAX, MAX, True), (2 ** 24, 255, False), (2 ** 24, 256, True)])
def test_recurrence_step(B, D, refused):
    assert code("hattn_gated_recurrence_step", *([None] * 4), B, D, FS, FS, None) == \
        (NOT if refused else VAL)


def attention(B, T, H, G, D, window, sinks, train):
    dims = (B, T, H, G, D, window, sinks, 1.0, BF)
    fwd = [None] * 7
    if train:
        fwd[6] = 16  # lse: a placeholder that no launch sees
    got = code("hattn_sliding_fwd", *fwd, *dims, None)
    if train:
        assert got == code("hattn_sliding_bwd", *([None] * 11), *dims, None, 0, None)
    return got


# a launch's workgroups come in eights
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("B,T,H,refused", [
    (2 ** 24 - 8, 1, 1, False), (2 ** 24 - 7, 1, 1, True), (2 ** 24 - 8, 128, 1, False),
    (2 ** 23 - 4, 129, 1, False), (2 ** 23 - 3, 129, 1, True), (2 ** 14, 1, 1024, True),
    (2 ** 14 - 1, 1, 1024, False), (1, 2 ** 30 - 1, 1, False), (1, 2 ** 30, 1, True),
    (2, 2 ** 30 - 129, 1, True), (MAX, MAX, 2 ** 20, True)])
def test_attention(B, T, H, refused, train):
    assert attention(B, T, H, 1, 8, 4, 0, train) == (NOT if refused else VAL)


def test_attention_backward_is_refused_before_its_forward():
    """Two blocks of sinks make the backward's launch larger than the forward's."""
    assert attention(2 ** 22, 100, 2, 1, 8, 4, 33, False) == VAL
    assert attention(2 ** 22, 100, 2, 1, 8, 4, 33, True) == NOT
    assert attention(2 ** 22 - 2, 100, 2, 1, 8, 4, 33, True) == VAL
    assert attention(2 ** 22, 100, 2, 1, 8, 4, 32, True) == VAL
    assert attention(2 ** 22, 100, 2, 1, 8, 100, 33, True) == VAL  # no query is far from a sink
    assert attention(2 ** 23, 100, 1, 1, 8, 4, 32, True) == NOT  # 2^32 values of the sinks' sums
    assert attention(2 ** 23, 100, 1, 1, 8, 4, 31, True) == VAL
    lib = _lib.load()
    assert lib.hattn_sliding_bwd_workspace(2 ** 22, 100, 2, 1, 8, 4, 33) == 0
    assert lib.hattn_sliding_bwd_workspace(2 ** 22 - 2, 100, 2, 1, 8, 4, 33) > 0
    assert lib.hattn_sliding_bwd_workspace(1, MAX, 1, 1, 8, 1, 4) == 0


# pieces of 8 values
@pytest.mark.parametrize("B,G,D,window,sinks,refused", [
    (1, 1, 8, MAX, 0, False), (1, 1, 8, MAX, 1, True), (2, 1, 8, MAX, 0, True), (2, 1, 8, MAX - 127, 0, False),
    (2, 1, 16, MAX, 0, True), (2 ** 16, 1, 8, 2 ** 16 - 1, 0, False), (2 ** 16, 1, 8, 2 ** 16 - 1, 1, True),
    (2 ** 16, 1, 8, 2 ** 16, 0, True), (MAX, 1, 128, MAX, 0, True)])
def test_cache_fill(B, G, D, window, sinks, refused):
    assert code("hattn_sliding_cache_fill", *([None] * 7), B, 4, G, D, window, sinks, BF, None) == \
        (NOT if refused else VAL)


@pytest.mark.parametrize("B,H,G,window,sinks,refused", [
    (2 ** 24 - 1, 1, 1, 4, 0, False), (2 ** 24, 1, 1, 4, 0, True), (2 ** 23, 17, 1, 4, 0, True),
    (2 ** 21, 16, 1, 4, 0, True), (2 ** 21 - 1, 16, 1, 4, 0, False), (2 ** 20, 32, 1, 4, 0, True), (2 ** 20 - 1, 32, 1, 4, 0, False),
    (1, 1, 1, MAX - 2 ** 14, 0, False), (1, 1, 1, MAX - 2 ** 14, 1, True), (1, 1, 1, MAX, 64, True),
    (MAX, 2 ** 20, 1, 4, 0, True)])
def test_step(B, H, G, window, sinks, refused):
    assert code("hattn_sliding_step", *([None] * 7), B, H, G, 8, window, sinks, 1.0, BF, None, 0,
                None) == (NOT if refused else VAL)
    if window > MAX - 2 ** 15:
        assert (_lib.load().hattn_sliding_step_workspace(B, H, G, 8, window, sinks) == 0) == refused
