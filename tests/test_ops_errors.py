"""GPU: an error of the runtime that an operator's C entry reports does not stay
behind, where the next check of the same thread (torch's after its next kernel)
would report it again.  A device that is not there is such an error."""
import ctypes as C

import pytest
import torch

from gene2vec_amd import _native as N

P = 0x10000  # a stand-in for an address: the device is looked for before it is used


def fail(device):
    L = N.lib()
    need = C.c_int64()
    one = (C.c_void_p * 1)(P), (C.c_int64 * 1)(4), (C.c_int32 * 1)(N.F32)
    yield L.g2v_embed_lookup(device, P, N.F32, 10, 4, 4, P, 8, 3, 1.0, P, N.F32, None)
    L.g2v_embed_grad_workspace(3, 10, 4, C.byref(need))
    yield L.g2v_embed_grad(device, P, N.F32, 4, P, 8, 3, 10, 4, 1.0, -1, P, N.F32, P, need, None)
    L.g2v_global_norm_workspace(1, C.byref(need))
    yield L.g2v_global_norm(device, *one, 1, P, P, need, None)
    yield L.g2v_clip_global_norm(device, one[0], one[0], *one[1:], 1, 1.0, P, P, need, None)


def check(device):
    left = N.lib().hipPeekAtLastError
    left.restype = C.c_int
    N.lib().hipGetLastError()
    for rc in fail(device):
        assert rc == N.G2V_EHIP and N.lib().g2v_last_error()
        assert left() == 0


@pytest.mark.gpu
def test_no_error_stays_behind():
    x = torch.ones(4, device="cuda")
    check(4096)
    assert float((x + 1).sum()) == 8.0
