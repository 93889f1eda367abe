"""Numbers of a stored computation that become enumerators or are multiplied on loading: values outside their range are refused."""
import ctypes
import struct

import numpy as np


def _fnv1a(data):
    h = 1469598103934665603
    for c in data:
        h = ((h ^ c) * 1099511628211) & (2 ** 64 - 1)
    return h


def _load(odla, body):
    L = odla.load_library()
    loc, keep = odla.memory_location(bytes(body) + struct.pack("<Q", _fnv1a(bytes(body))))
    comp = ctypes.c_void_p()
    L.odla_SetLogLevel(0)
    st = L.odla_LoadComputation(loc, ctypes.byref(comp))
    L.odla_SetLogLevel(2)
    if st == 0:
        assert L.odla_DestroyComputation(comp) == 0
    return st


def test_precision_mode_and_extents_are_checked(odla, tmp_path):
    path = str(tmp_path / "relu.odla")
    hb = odla.HipBuilder()
    try:
        hb.output(hb.relu(hb.arg("x", (1234567, 7654321)), name="y"), "y")
        loc, keep = odla.path_location(path)
        assert hb.L.odla_StoreComputation(loc, hb.comp) == 0
    finally:
        hb.destroy()
    body = bytearray(open(path, "rb").read()[:-8])
    assert _load(odla, body) == 0
    for mode in (-1, 4, 1 << 24, 1 << 40):                 # the second number behind the signature
        bad = bytearray(body)
        struct.pack_into("<q", bad, 16, mode)
        assert _load(odla, bad) == odla.ODLA_INVALID_PARAM
    at = body.index(struct.pack("<qq", 1234567, 7654321))
    for extents in ((0, 1), (-1, -1), (1 << 40, 1), ((1 << 32) + 3, (1 << 32) - 1), (1 << 39, 1 << 39)):
        bad = bytearray(body)
        struct.pack_into("<qq", bad, at, *extents)
        assert _load(odla, bad) == odla.ODLA_INVALID_PARAM
