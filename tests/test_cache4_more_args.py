"""More of what the 4-bit cache's calls refuse before touching a device (CPU
only); the helpers are test_cache4_args'."""
import ctypes

import pytest

import libpktito_b200 as P
from tests import test_cache4_args as A

EINVAL = A.EINVAL


def append_if(status, **kw):
    a = dict(layer=1, k=A.A, ks=128, v=A.A, vs=128, type=P.F32, seqs=A.A, starts=A.A, n=2, rows=4)
    a.update(kw)
    return P.lib().pkb_cache4_append_if_dev(0, ctypes.byref(A.cache()), *a.values(), status)


def test_append_after_a_page_operation_refuses_what_append_does():
    assert append_if(A.A + 2) == append_if(A.A, layer=2) == append_if(A.A, k=None) == append_if(None, ks=127) == EINVAL
    assert append_if(A.A, n=0) == append_if(None, rows=0) == 0


def test_append_checks_its_status():
    import torch
    c = P.Cache4.of(torch.zeros((1, 5, P.cache4_page_bytes(16, 2, 32)), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.int32),
                    torch.zeros(3, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), 16, 2, 32)
    good, rows = torch.zeros(4, dtype=torch.int32), torch.zeros((4, 64))
    for bad in (good.long(), good[:0], good.float()):
        with pytest.raises(P.PkbError, match="int32"):
            P.cache4_append_dev(c, 0, rows, 64, rows, 64, good, good, 2, 4, 0, status=bad)
