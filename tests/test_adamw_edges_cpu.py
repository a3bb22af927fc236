"""CPU checks of the AdamW operators at their edges: refusals of the row-aware gradient norm."""
import ctypes


def _one(*x):
    return (ctypes.c_void_p * 1)(*x)


def test_norm_without_rows_that_are_left_alone_refuses_before_it_launches():
    from gs_icp_slam_amd import _lib
    lib = _lib.load()
    width, frozen = (ctypes.c_int * 1)(3), (ctypes.c_int * 1)(1)
    D = _lib.AdamWDevice

    def norm(d, grad=64, numel=300, dtype=0, n=1, out=64, scratch=64):
        return lib.gsicp_grad_norm_rows(n, _one(grad), (ctypes.c_longlong * 1)(numel), (ctypes.c_int * 1)(dtype), ctypes.addressof(d) if d else None, 1.0, out, 64, scratch, None)
    w, f = ctypes.addressof(width), ctypes.addressof(frozen)
    ok = dict(live_rows=64, row_width=w, row_freeze=64, group_frozen=f)
    assert norm(None) == -2
    assert norm(D(live_rows=64)) == -2                                            # no row_width
    assert norm(D(row_width=w, row_freeze=64)) == -2                              # no group_frozen
    assert norm(D(grad_rows=64, **ok)) == -2                                      # gradients that were not written
    assert norm(D(**ok), dtype=1) == -2 and norm(D(**ok), numel=1 << 32) == -2    # as in the step
    assert norm(D(**ok), numel=-1) == -2 and norm(D(**ok), numel=(1 << 33) + 1) == -2 and norm(D(**ok), dtype=3) == -2
    assert norm(D(**ok), grad=0) == -2 and norm(D(**ok), grad=1 << 58) == -2 and norm(D(**ok), out=None) == -2 and norm(D(**ok), n=-1) == -2
    assert norm(D(**ok), numel=1 << 30, scratch=None) == -2
    assert b"gsicp_grad_norm" in lib.gsicp_last_error()
