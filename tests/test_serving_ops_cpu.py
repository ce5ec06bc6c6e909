"""Argument checks of the serving operators that need no device."""
import ctypes

import pytest


def _jobs(*shapes):
    import rsv
    return (rsv.AdapterJob * len(shapes))(*[rsv.AdapterJob(0, 0, n, k, 0, 0, 0, e) for n, k, e in shapes])


def test_adapter_work_limits():
    import rsv
    lib = rsv.hip_lib()
    ok = _jobs((2560, 2560, 0), (64, 8, 3))
    assert lib.rsv_adapter_work(ok, 2, 16, 64) > 0
    assert lib.rsv_adapter_work(ok, 2, 128, 1 << 20) > 0
    for jobs, njobs, rank, rows, text in [
            (ok, 0, 16, 64, b"jobs"), (ok, 9, 16, 64, b"jobs"), (None, 1, 16, 64, b"jobs"), (ok, 2, 0, 64, b"rank"),
            (ok, 2, 4, 64, b"rank"), (ok, 2, 20, 64, b"rank"), (ok, 2, 136, 64, b"rank"), (ok, 2, 16, 0, b"rows"),
            (ok, 2, 16, (1 << 20) + 1, b"rows"), (_jobs((2564, 64, 0)), 1, 16, 1, b"multiples of 8"),
            (_jobs((64, 0, 0)), 1, 16, 1, b"multiples of 8"), (_jobs((64, 1 << 25, 0)), 1, 16, 1, b"multiples of 8"),
            (_jobs((64, 64, 1)), 1, 16, 1, b"epilogue")]:
        assert lib.rsv_adapter_work(jobs, njobs, rank, rows) == 0
        assert text in lib.rsv_last_error()


def test_logits_work_limits():
    import rsv
    lib = rsv.hip_lib()
    for n, rows in ((0, 1), (1048577, 1), (65536, 0), (65536, (1 << 20) + 1)):
        assert lib.rsv_logits_work(n, rows) == 0
        assert b"logits_work" in lib.rsv_last_error()


@pytest.mark.parametrize("name,nargs", [("rsv_adapter_multi", 9), ("rsv_sample_rand_batch", 8),
                                        ("rsv_token_logprobs", 7), ("rsv_store_filter", 6)])
def test_null_context(name, nargs):
    import rsv
    fn = getattr(rsv.hip_lib(), name)
    args = [None if t is ctypes.c_void_p else t(1) for t in fn.argtypes[1:]]
    assert len(args) == nargs
    assert fn(None, *args) != 0
    assert b"null context" in rsv.hip_lib().rsv_last_error()


def test_logits_pieces_limit():
    """A block takes a piece of 8192: more than 2^22 pieces are refused, that many are not."""
    import rsv
    lib = rsv.hip_lib()
    assert lib.rsv_logits_work(65536, 1 << 19) > 0
    assert lib.rsv_logits_work(65536, (1 << 19) + 1) == 0
    assert b"pieces" in lib.rsv_last_error()
    assert lib.rsv_logits_work(8193, 1 << 20) > 0 and lib.rsv_logits_work(1048576, 1 << 20) == 0
