"""The pair-averaging model store's shared headers (parallel/kungfu.py)."""

import os
import uuid

import pytest

from kf_benchmarks_amd.ops import _native as N
from kf_benchmarks_amd.parallel import kungfu


@pytest.mark.parametrize("refused", [True, False])
def test_header_is_unmapped_only_once_unregistered(monkeypatch, refused):
    """A mapping that the device may still read (its unregistering failed) stays mapped when the header is closed."""
    header = kungfu._Header("test_%s" % uuid.uuid4().hex, 0, 1)
    header.write(0, 6)
    m = header._map(0)
    calls = []

    def call(name, *args):
        calls.append(name)
        if name == "kfb_host_register":
            args[2]._obj.value = 4096
        elif refused:
            raise N.NativeError("refused")
        return 0

    monkeypatch.setattr(N, "call", call)
    assert header.device_word(0, 1) == 4104
    held = len(kungfu._Header._held)
    header.close()
    assert calls == ["kfb_host_register", "kfb_host_unregister"]
    assert m.closed == (not refused) and len(kungfu._Header._held) == held + refused
    assert not os.path.exists(header.paths[0])
    if refused:
        assert m[:1] == b"\x06"
