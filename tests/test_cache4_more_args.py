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


def small():
    import torch
    return P.Cache4.of(torch.zeros((1, 5, P.cache4_page_bytes(16, 2, 32)), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.int32),
                       torch.zeros(3, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), 16, 2, 32)


def short_rows():
    """Tensors that do not hold 4 rows of 64 values, 80 values apart."""
    import torch
    x = torch.zeros((8, 160))
    return [x[:2, :80], x[:4, :63], x[:2, :80].flatten()[:303], x[:4, :128:2], x[:4].t(), x[4:, :0], x[:4, :80].t().contiguous().t(),
            x[:4].view(4, 4, 40)[:, :2, :32], x[7:, 100:], x[:1, :64].expand(4, 64)]


@pytest.mark.parametrize("at", range(10))
def test_calls_check_that_tensors_hold_their_rows(at):
    import torch
    c, n, bad, good = small(), torch.zeros(4, dtype=torch.int32), short_rows()[at], torch.zeros((4, 80))
    work = torch.zeros(1 << 16, dtype=torch.uint8)
    for a, b in ((bad, good), (good, bad)):
        for call in (lambda: P.cache4_append_dev(c, 0, a, 80, b, 80, n, n, 2, 4, 0), lambda: P.cache4_read_dev(c, 0, a, 80, b, 80, n, n, 2, 4, 0),
                     lambda: P.attention_cache4_dev(a, 80, b, 80, 2, c, 0, n, n, 2, 4, 4, 0.1, True, 0, work, 0)):
            with pytest.raises(P.PkbError, match="4 rows of 64 values"):
                call()


def test_tensors_that_hold_their_rows_pass():
    # as far as the device, which is not there
    import torch
    c, n, work = small(), torch.zeros(4, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)
    x = torch.zeros((8, 160))
    good = [x[:4], x[:4, 80:], x[:4, :64], x.view(8, 5, 32)[:4, 1:3], x.flatten()[:3 * 160 + 64], x[:4, None, :64], x.view(16, 80)[::2][:4, :64]]
    if torch.cuda.is_available():
        pytest.skip("host memory is no place for a device's rows")
    for a in good:
        b = torch.zeros((4, 160))
        for call in (lambda: P.cache4_append_dev(c, 0, a, 160, b, 160, n, n, 2, 4, 0), lambda: P.cache4_read_dev(c, 0, a, 160, b, 160, n, n, 2, 4, 0),
                     lambda: P.cache4_append_dev(c, 0, a[:1] if a.dim() > 1 else a, 1, b[:1], 0, n, n, 1, 1, 0)):
            with pytest.raises(P.PkbError) as e:
                call()
            assert "ENODEV" in str(e.value), (a.shape, a.stride(), e.value)


@pytest.mark.parametrize("stream", [None, 0])
def test_a_cache_on_another_device_than_the_current_one_is_refused(stream, monkeypatch):
    import torch
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    c, n, x, work = small(), torch.zeros(4, dtype=torch.int32), torch.zeros((4, 64)), torch.zeros(1 << 16, dtype=torch.uint8)
    for c.device in (-1, 1):  # host memory; a second GPU
        for call in (lambda: P.cache4_reset_dev(c, stream), lambda: P.cache4_grow_dev(c, n, n, 2, n, work, stream),
                     lambda: P.cache4_fork_dev(c, n, n, n, 2, n, work, stream), lambda: P.cache4_free_dev(c, n, 2, n, work, stream),
                     lambda: P.cache4_copy_dev(c, c, n, n, n, 2, n, work, stream), lambda: P.cache4_compact_dev(c, None, n, work, stream),
                     lambda: P.cache4_append_dev(c, 0, x, 64, x, 64, n, n, 2, 4, stream),
                     lambda: P.cache4_read_dev(c, 0, x, 64, x, 64, n, n, 2, 4, stream),
                     lambda: P.attention_cache4_dev(x, 64, x, 64, 2, c, 0, n, n, 2, 4, 4, 0.1, True, 0, work, stream)):
            with pytest.raises(P.PkbError, match="a cache on device"):
                call()


def test_a_copy_between_devices_is_refused():
    import torch
    c, to, n, work = small(), small(), torch.zeros(4, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)
    to.device = 1
    with pytest.raises(P.PkbError, match="caches on devices"):
        P.cache4_copy_dev(to, c, n, n, n, 2, n, work, 0)


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) - 1])
def test_lists_past_what_is_counted_in_32_bits_are_refused(n):
    one = A.cache(n_heads=1)
    assert A.rows(one, n=n) == A.rows(one, append=False, n=n) == A.attend(one, H=1, n=n) == EINVAL
