"""The tile rule of the bf16 products (csrc/q38m_linear_tiles.h) as the tests ask
it: a host library built once a run."""
import collections
import ctypes
import functools
import os
import subprocess
import tempfile

from conftest import PACKAGE_DIR

Tiles = collections.namedtuple("Tiles", "rows columns parts each at_most workgroups held waves")


@functools.lru_cache(None)
def _library():
    folder = tempfile.TemporaryDirectory(prefix="linear_tiles_")
    path = os.path.join(folder.name, "linear_tiles.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PACKAGE_DIR, "csrc"), "-o", path,
                    os.path.join(os.path.dirname(os.path.abspath(__file__)), "linear_tiles_check.cpp")], check=True)
    lib = ctypes.CDLL(path)
    lib.linear_tiles_of.argtypes = [ctypes.c_uint32] * 8 + [ctypes.c_void_p]
    lib.linear_tiles_of.restype = None
    return lib, folder


def tiles_of(rows, columns, depth, experts=0, swiglu=False, ragged=False, wide=True, along=False):
    """rows and columns of C (in front of a fold), depth: K; ragged: weights' gradients; along:
    forward products."""
    result = (ctypes.c_uint32 * 8)()
    _library()[0].linear_tiles_of(rows, columns, depth, experts, swiglu, ragged, along, wide, result)
    return Tiles(*result)


SHAPES = {(256, 256), (128, 128), (64, 64), (32, 128), (16, 128)}
FEW = {(16, 16, 8), (16, 32, 8), (16, 32, 4)}  # rows, columns, waves
