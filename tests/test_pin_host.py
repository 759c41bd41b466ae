"""The payload ring's registration as pinned memory, where the system refuses it (no GPU is touched)."""
import pytest
import torch

from aiforearth_api_platform_amd.ops import _ext
from aiforearth_api_platform_amd.runtime import gpu_worker


class Library:
    """A kernel library; ``cleared`` counts the calls that clear a pending error."""

    cleared = 0

    def ai4e_clear_error(self):
        self.cleared += 1
        return 801


@pytest.fixture
def register(monkeypatch):
    def use(answer, library):
        class Runtime:
            def cudaHostRegister(self, ptr, size, flags):
                if isinstance(answer, Exception):
                    raise answer
                return answer

        monkeypatch.setattr(torch.cuda, "cudart", Runtime)
        monkeypatch.setattr(_ext, "available", lambda: library is not None)
        monkeypatch.setattr(_ext, "lib", lambda: library)
        return gpu_worker.pin_host(torch.zeros(16, dtype=torch.uint8))

    return use


@pytest.mark.parametrize("answer", [801, (801,)])
def test_a_refusal_leaves_no_error(register, answer):
    library = Library()
    assert register(answer, library) is False and library.cleared == 1


@pytest.mark.parametrize("answer", [0, (0,), RuntimeError("no runtime")])
def test_other_errors_stay(register, answer):
    """Registered, or not called at all: an error that is pending then is another call's."""
    library = Library()
    assert register(answer, library) is (not isinstance(answer, Exception)) and library.cleared == 0


@pytest.mark.parametrize("library", [None, object()])
def test_a_refusal_with_a_library_that_cannot_clear(register, library):
    """No kernel library, or one of an older tree: the ring stays pageable, the worker goes on."""
    assert register(801, library) is False
