"""The tile rule of the microscaled products (csrc/q38m_mx_tiles.h) as the
tests ask it: a host library built once a run."""
import collections
import ctypes
import functools
import os
import subprocess
import tempfile

import numpy as np

from conftest import PACKAGE_DIR

Tiles = collections.namedtuple("Tiles", "rows columns wide streamed at_most workgroups")


@functools.lru_cache(None)
def _library():
    folder = tempfile.TemporaryDirectory(prefix="mx_tiles_")
    path = os.path.join(folder.name, "mx_tiles.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PACKAGE_DIR, "csrc"), "-o", path,
                    os.path.join(os.path.dirname(os.path.abspath(__file__)), "mx_tiles_check.cpp")], check=True)
    lib = ctypes.CDLL(path)
    lib.mx_tiles_of.argtypes = [ctypes.c_uint32] * 6 + [ctypes.c_void_p]
    lib.mx_tiles_of.restype = None
    return lib, folder


def tiles_of(routes, n, columns, experts=0, swiglu=False, scales_aligned=True):
    """experts 0: the dense product of `routes` rows by n."""
    result = (ctypes.c_uint32 * 6)()
    _library()[0].mx_tiles_of(routes, n, columns, experts, swiglu, scales_aligned, result)
    return Tiles(*result)


def count(tiles, n, swiglu, offsets):
    """Tiles of a routing: row tiles of each expert's rows times tiles across."""
    across = tiles.columns // 2 if swiglu else tiles.columns
    rows = np.diff(np.asarray(offsets, np.int64))
    return int((-(-rows // tiles.rows)).sum()) * (-(-(n // 2 if swiglu else n) // across))
