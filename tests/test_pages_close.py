"""Closing the owners of a handle (capi.Blit, capi.Pages) where the library refuses: what
it has left alive stays reachable, and can be closed later."""
import pytest


class _Answers:
    """Stands for the library: the next statuses of the two destroy calls."""

    def __init__(self, *statuses):
        self.statuses, self.handles = list(statuses), []

    def _destroy(self, handle):
        self.handles.append(handle)
        return self.statuses.pop(0)

    mi355_blit_destroy = mi355_blit_pages_destroy = _destroy


@pytest.fixture(scope="module")
def capi_host(pkg):
    import torch  # noqa: F401  (one HIP runtime per process: torch's first)
    pkg.capi.load()
    return pkg.capi


def _owner(cls, lib):
    owner = cls.__new__(cls)
    owner.lib, owner.handle = lib, 16
    return owner


@pytest.mark.parametrize("what", ["Blit", "Pages"])
def test_a_refused_close_keeps_the_handle(capi_host, what):
    lib = _Answers(capi_host.ERROR_INVALID_ARGUMENT, capi_host.SUCCESS)
    owner = _owner(getattr(capi_host, what), lib)
    with pytest.raises(capi_host.BlitError) as e:
        owner.close()
    assert e.value.status == capi_host.ERROR_INVALID_ARGUMENT
    owner.close()
    owner.close()  # closed: nothing is destroyed twice
    assert lib.handles == [16, 16] and owner.handle is None


def test_an_engine_that_went_with_an_error_is_gone(capi_host):
    """Every answer of mi355_blit_destroy but INVALID_ARGUMENT is that of a freed handle."""
    lib = _Answers(capi_host.ERROR)
    owner = _owner(capi_host.Blit, lib)
    with pytest.raises(capi_host.BlitError):
        owner.close()
    owner.close()
    assert lib.handles == [16]


def test_a_pool_that_could_not_be_waited_for_stays(capi_host):
    """mi355_blit_pages_destroy frees nothing unless it succeeds."""
    lib = _Answers(capi_host.ERROR, capi_host.SUCCESS)
    owner = _owner(capi_host.Pages, lib)
    with pytest.raises(capi_host.BlitError):
        owner.close()
    owner.close()
    assert lib.handles == [16, 16]


@pytest.mark.gpu
def test_an_engine_with_an_open_pool_is_closed_after_the_pool(torch_cuda, capi):
    buf = torch_cuda.zeros(4096, dtype=torch_cuda.uint8, device="cuda:0")
    blit = capi.Blit(0)
    pool = capi.Pages(blit, [(buf.data_ptr(), 64, 16, 1)], 4, 4)
    with pytest.raises(capi.BlitError) as e:
        blit.close()
    assert e.value.status == capi.ERROR_INVALID_ARGUMENT
    # both work as before
    assert blit.fill32(buf.data_ptr(), 7, 16) == capi.SUCCESS and blit.synchronize() == capi.SUCCESS
    assert int(buf.sum()) == 7 * 16
    pool.close()
    blit.close()
    assert blit.handle is None
