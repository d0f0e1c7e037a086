"""CPU: what the entry points of packed sequences refuse at their edges."""
import ctypes as C


def test_what_rounding_left_is_only_there_beside_the_statistics(built_library):
    """A forward without lse leaves no o_rest: asking for it is an error, not memory as it was.  (Addresses are made up: the call
    does not get as far as a launch.)"""
    from evoformer_triton_b200 import _lib
    lib = _lib.load()
    for more in (dict(), dict(key_offsets=256), dict(key_offsets=256, key_form=1), dict(dtype=2), dict(flags=_lib.FLAG_FORCE_GENERIC)):
        p = _lib.PackedParams(B=2, H=4, Hk=2, D=64, Tq=10, Tk=10, scale=1.0, q=256, k=256, v=256, o=256, offsets=256, o_rest=512, **more)
        assert lib.evoattn_packed_fwd(C.byref(p), None) == 1 and lib.evoattn_packed_fwd_workspace_bytes(C.byref(p)) == 0
