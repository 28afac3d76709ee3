"""Memory that ends, or begins, where nothing may be touched."""
import ctypes
import mmap

import numpy as np

PAGE = mmap.PAGESIZE
libc = ctypes.CDLL(None, use_errno=True)
libc.mmap.restype = ctypes.c_void_p
libc.mmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_long]
libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
libc.munmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t]


class Guarded:
    """n bytes between two pages that cannot be touched, at the end of what lies between them or at its beginning."""

    def __init__(self, n, at_end=True, align=1):
        inner = max(-(-n // PAGE), 1) * PAGE
        self.size = inner + 2 * PAGE
        self.base = libc.mmap(None, self.size, 3, 0x22, -1, 0)          # private, anonymous
        assert self.base not in (None, ctypes.c_void_p(-1).value)
        for page in (self.base, self.base + PAGE + inner):
            assert libc.mprotect(page, PAGE, 0) == 0
        assert not at_end or n % align == 0
        self.at, self.n = self.base + PAGE + (inner - n if at_end else 0), n
        ctypes.memset(self.base + PAGE, 0xA5, inner)

    def array(self, dtype):
        return np.frombuffer((ctypes.c_char * self.n).from_address(self.at), dtype)

    def __del__(self):
        libc.munmap(self.base, self.size)


def guarded(a, at_end=True):
    if a is None:
        return None
    a = np.ascontiguousarray(a)
    g = Guarded(a.nbytes, at_end)
    g.array(a.dtype)[:] = a.ravel()
    return g
