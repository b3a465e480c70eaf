"""The dense operators' status word: no report is lost between readers and
the streams that set bits."""
from __future__ import annotations

import ctypes
import threading

import pytest
import torch


class _Word:
    """The device word as an array that torch can alias."""

    def __init__(self, address):
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (address, False), "version": 3}


def _word():
    import ffn_host

    address = ctypes.c_void_p()
    assert ffn_host._library().moe_b200_dense_status_address(ctypes.byref(address)) == 0
    return torch.as_tensor(_Word(address.value), device="cuda")


@pytest.mark.gpu
def test_read_takes_what_is_set(cuda_device):
    import ffn_host

    word = _word()
    assert ffn_host.read_status() == 0
    for bits in (1, 2, 4, 7):
        word.fill_(bits)
        assert ffn_host.read_status() == bits
        assert ffn_host.read_status() == 0 and word.item() == 0
    status = ctypes.c_uint32(5)
    stream = torch.cuda.current_stream().cuda_stream
    assert ffn_host._library().moe_b200_dense_read_status(ctypes.byref(status), stream) == 0 and status.value == 0
    word.fill_(2)
    torch.cuda.synchronize()
    assert ffn_host._library().moe_b200_dense_read_status(ctypes.byref(status), stream) == 7 and status.value == 2


@pytest.mark.gpu
def test_a_report_during_a_read_is_kept(cuda_device):
    """Another stream sets a bit at any time around a read: that read or the
    next reports it."""
    import ffn_host

    word = _word()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert ffn_host.read_status() == 0
    lost = 0
    for n in range(400):
        start = threading.Barrier(2)

        def report():
            start.wait()
            with torch.cuda.stream(side):
                for _ in range(n % 8):
                    torch.cuda._sleep(2000)          # a few microseconds later each time
                word.fill_(4)
            side.synchronize()

        t = threading.Thread(target=report)
        t.start()
        start.wait()
        seen = 0
        while t.is_alive():
            seen |= ffn_host.read_status()
        t.join()
        seen |= ffn_host.read_status()
        lost += seen != 4
    assert lost == 0
    assert ffn_host.read_status() == 0


def test_address_refusal():
    import ffn_host

    assert ffn_host._library().moe_b200_dense_status_address(None) == 1
