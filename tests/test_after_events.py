"""Receiver.after (foa_rx_after from Python): the library keeps raw event handles, so the receiver keeps the event objects alive -- all of
them, up to the sixteen the library takes -- until the call that waits for them is back, and lets them go then.  No GPU: the C ABI is a stand-in
that follows the library's rules and looks at which events are alive when it is called."""
import gc
import weakref

import numpy as np
import pytest

import fun_ofdm_amd as foa
from fun_ofdm_amd import rx as rx_mod


class Event:
    """what Receiver uses of a torch.cuda.Event; destroyed with its last reference"""
    made = 0

    def __init__(self):
        Event.made += 1
        self.cuda_event = 0x1000 + Event.made

    def record(self, stream=None):
        self.stream = stream


class Abi:
    """foa_rx_after and the calls that take its events; rc: what those calls return"""

    def __init__(self):
        self.handles, self.alive, self.rc, self.seen = [], weakref.WeakValueDictionary(), 0, []

    def track(self, ev):
        self.alive[ev.cuda_event] = ev
        return ev

    def foa_rx_after(self, h, handle):
        if len(self.handles) >= 16:
            return -5
        self.handles.append(handle)
        return 0

    def foa_last_error(self):
        return b"refused by the stand-in"

    def foa_tx_build_frames_dev(self, h, payloads, pitch, length, rate, n, out, got):
        if n == 0:                                            # (the size query takes nothing)
            got._obj.value = 480
            return 0
        return self.taking("foa_tx_build_frames_dev")

    def foa_rx_sync(self, h):
        return 0

    def taking(self, name):
        gc.collect()
        dead = [x for x in self.handles if x not in self.alive]
        self.seen.append((name, len(self.handles), len(dead)))
        self.handles = []
        return self.rc

    def __getattr__(self, name):
        if name.startswith("foa_rx_destroy") or name.startswith("foa_stream_destroy"):
            return lambda *a: None
        return lambda *a: self.taking(name)


@pytest.fixture
def receiver():
    r = object.__new__(foa.Receiver)
    r._lib, r._h, r.device, r._after_keep = Abi(), 1, 0, []
    return r


class Stream:
    def __init__(self, idle):
        self.idle = idle

    def query(self):
        return self.idle


@pytest.fixture
def busy_torch(monkeypatch, receiver):
    import torch
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(False))
    monkeypatch.setattr(torch.cuda, "Event", lambda *a, **k: receiver._lib.track(Event()))
    return torch


def calls(r, torch):
    iq, d, e = np.zeros(400, np.complex64), np.zeros(2, foa.frame_desc_dtype), np.zeros(2, np.int64)
    tq, td, te = torch.zeros(400, dtype=torch.complex64), torch.zeros(96, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64)
    tp, tr = torch.zeros((2, 64), dtype=torch.uint8), torch.zeros((2, 4), dtype=torch.int32)
    return {"decode_frames_host": (0, lambda: r.decode_frames_host(iq, d, e)),
            "decode_frames_f64_host": (0, lambda: r.decode_frames_f64_host(iq, d, e)),
            "submit_host": (0, lambda: r.submit_host(iq, d, e)),
            "decode_frames_dev": (1, lambda: r.decode_frames_dev(tq, td, te, tp, tr)),
            "decode_frames_dev, settled": (0, lambda: r.decode_frames_dev(tq, td, te, tp, tr, settle=False)),
            "sync_dev": (1, lambda: r.sync_dev(tq, td, te)),
            "sync_dev_begin": (1, lambda: r.sync_dev_begin(tq, td, te)),
            "tx_channel": (1, lambda: r.tx_channel(torch.zeros((1, 480, 2), dtype=torch.float64), 600, 10, 25.0, 1)),
            "Stream": (0, lambda: rx_mod.Stream(r, 4096))}


@pytest.mark.parametrize("rc", [0, -1])
@pytest.mark.parametrize("name", ["decode_frames_host", "decode_frames_f64_host", "submit_host", "decode_frames_dev", "decode_frames_dev, settled", "sync_dev",
                                  "sync_dev_begin", "tx_channel", "Stream"])
def test_every_registered_event_lives_until_the_call_is_back(receiver, busy_torch, name, rc):
    abi = receiver._lib
    for n in (1, 2, 15):
        own, call = calls(receiver, busy_torch)[name]          # own: the event of torch's current stream, registered by the wrapper itself
        for _ in range(n):
            receiver.after(abi.track(Event()))                 # (no reference of the caller's is left)
        gc.collect()
        assert len(abi.alive) == n
        abi.rc, abi.seen = rc, []
        if rc:
            with pytest.raises(foa.FoaError):
                call()
        else:
            call()
        assert [s[1:] for s in abi.seen] == [(n + own, 0)], abi.seen
        gc.collect()
        assert len(abi.alive) == 0 and not receiver._after_keep          # ... and no longer than that


def test_building_frames_waits_although_it_asks_for_their_size_first(receiver, busy_torch):
    abi = receiver._lib
    receiver.after(abi.track(Event()))
    receiver.after(abi.track(Event()))
    pay = busy_torch.zeros((1, 10), dtype=busy_torch.uint8)

    class OnDevice:                                            # (the wrapper insists on a device tensor)
        is_cuda, dtype, shape, device = True, pay.dtype, pay.shape, pay.device
        dim, stride, data_ptr = staticmethod(pay.dim), staticmethod(pay.stride), staticmethod(pay.data_ptr)

    receiver.tx_build_frames(OnDevice(), 10)
    assert abi.seen == [("foa_tx_build_frames_dev", 3, 0)]
    gc.collect()
    assert len(abi.alive) == 0


def test_an_event_the_library_refuses_is_not_kept(receiver):
    abi = receiver._lib
    for _ in range(16):
        receiver.after(abi.track(Event()))
    with pytest.raises(foa.FoaError):
        receiver.after(abi.track(Event()))
    gc.collect()
    assert len(abi.alive) == 16
