"""Result arrays in page-locked host memory, recycled.

The reference returns freshly allocated numpy arrays (``dosma/core/fitting.py:205-215``: ``np.full`` + scatter).  On the
GPU path a fresh 0.7 GB result costs more than the fit: the operating system zero-fills every page on first touch
(65 ms per GB on the benchmark host) and the download has to go through a staging buffer.  Here large
results live in ``hipHostMalloc`` memory handed out by ``empty()``: the pages are resident and the copy is a true DMA.  A
block goes back to the free list when the last numpy view of it is garbage-collected (a ``weakref`` finalizer on the
exporting buffer object), so callers own their results exactly as before; nothing is ever overwritten under them.

``DOSMA_AMD_HOST_POOL_GB`` (default 8; 0 switches the pool off) bounds ALL page-locked bytes of the pool -- blocks on the
free list plus blocks still owned by live results (pinned memory cannot be swapped); beyond it ``empty()`` hands out plain
numpy arrays.  ``DOSMA_AMD_HOST_POOL=0`` switches the pool off as well.

Fork: ROCm maps page-locked allocations so that a ``fork()``ed child does not inherit them.  Blocks of ordinary memory are made
inheritable again by the library (``qmri_host_alloc``: ``madvise(MADV_DOFORK)``).  Where the runtime maps them from the device's
file instead (``HSA_USERPTR_FOR_PAGED_MEM=0``) the kernel refuses that for the mapping's kind (EINVAL), and nothing lies at the
block's address in the child: then ``os.fork`` puts an ordinary copy of every block that a live result holds there (the copy is
made before the fork, of live blocks only; the parent keeps none of it).  Either way a ``multiprocessing`` worker forked while
results are alive can READ them (tests/test_hostpool.py::test_forked_child_reads_a_pooled_result); a child never frees or recycles
the parent's blocks.
"""
import atexit
import ctypes
import gc
import os
import threading
import weakref

import numpy as np

_MIN_BYTES = 1 << 20        # smaller arrays: plain numpy
_GRANULE = 2 << 20          # size classes of 2 MB
_lock = threading.RLock()   # re-entrant: a finalizer (_release) can run inside a garbage collection that an allocation under
                            # the lock triggers on the same thread
_free = {}                  # size -> [pointers]
_cached = 0                 # bytes on the free list
_live = 0                   # bytes handed out and not yet released
_closed = False
_pid = os.getpid()          # blocks belong to the process that allocated them (a forked worker never frees or reuses them)
_held = {}                  # blocks of live results: pointer -> bytes
_apart = set()              # blocks a forked child does not inherit
_copies = []                # during a fork: (block, its copy, bytes)

# <sys/mman.h> of Linux
_PROT_RW, _MAP_PRIVATE_ANON, _MREMAP_MOVE_FIXED, _MADV_DOFORK = 0x3, 0x22, 0x3, 11
_libc = ctypes.CDLL(None, use_errno=True)
_libc.mmap.restype = ctypes.c_void_p
_libc.mmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_long]
_libc.munmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t]
_libc.mremap.restype = ctypes.c_void_p
_libc.mremap.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p]
_libc.madvise.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]


def _inherited(ptr, size):
    """Whether a forked child has the block (asked after the library has tried to make it so)."""
    return _libc.madvise(ptr, size, _MADV_DOFORK) == 0


def _before_fork():
    _lock.acquire()  # (no other thread gives a block back, or takes one, before the child has its copies)
    if _closed or os.getpid() != _pid or not _apart:
        return
    collects = gc.isenabled()
    gc.disable()         # (nor does a finalizer on this one)
    try:
        for ptr, size in _held.items():
            if ptr in _apart:
                to = _libc.mmap(None, size, _PROT_RW, _MAP_PRIVATE_ANON, -1, 0)
                if to not in (None, ctypes.c_void_p(-1).value):  # (no memory for it: the child is without this block)
                    ctypes.memmove(to, ptr, size)
                    _copies.append((ptr, to, size))
    finally:
        if collects:
            gc.enable()


def _after_fork_parent():
    while _copies:
        _, to, size = _copies.pop()
        _libc.munmap(to, size)
    _lock.release()


def _after_fork_child():
    while _copies:
        ptr, to, size = _copies.pop()
        _libc.mremap(to, size, size, _MREMAP_MOVE_FIXED, ptr)  # (the pages move, no second copy)
    _lock.release()


os.register_at_fork(before=_before_fork, after_in_parent=_after_fork_parent, after_in_child=_after_fork_child)


def _cap():
    try:
        return int(float(os.environ.get("DOSMA_AMD_HOST_POOL_GB", "8")) * (1 << 30))
    except ValueError:
        return 8 << 30


def _release(ptr, size):
    global _cached, _live
    if _closed or os.getpid() != _pid:  # interpreter shutdown / forked child: leave the block alone
        return
    cap = _cap()
    with _lock:
        _live -= size
        _held.pop(ptr, None)
        if _cached + _live + size <= cap:
            lst = _free.get(size)
            if lst is None:
                lst = _free[size] = []
            lst.append(ptr)
            _cached += size
            return
    try:
        from dosma_amd import _lib
        _apart.discard(ptr)
        _lib.load().qmri_host_free(ctypes.c_void_p(ptr))
    except Exception:       # pragma: no cover - nothing sensible to do in a finalizer
        pass


def _take(size):
    global _cached, _live
    with _lock:
        lst = _free.get(size)
        if lst:
            _cached -= size
            _live += size
            return lst.pop()
    return None


def empty(shape, dtype):
    """``numpy.empty(shape, dtype)`` in page-locked memory (plain numpy for small arrays, without a GPU, or when the
    allocation fails)."""
    global _live, _cached
    dt = np.dtype(dtype)
    shape = (shape,) if np.isscalar(shape) else tuple(int(s) for s in shape)
    count = 1
    for s in shape:
        count *= s
    nbytes = count * dt.itemsize
    cap = _cap()
    if (nbytes < _MIN_BYTES or _closed or cap <= 0 or os.getpid() != _pid
            or os.environ.get("DOSMA_AMD_HOST_POOL", "1") == "0"):
        return np.empty(shape, dt)
    size = (nbytes + _GRANULE - 1) // _GRANULE * _GRANULE
    ptr = _take(size)
    if ptr is None:
        with _lock:
            fits = _live + size <= cap
            drop = []
            if fits:
                _live += size  # reserved under the same lock as the check: concurrent callers cannot pass it together
                # make room among the cached blocks of other sizes first: the total stays below the cap
                for sz in sorted(_free, reverse=True):
                    while _free[sz] and _live + _cached > cap:
                        drop.append((sz, _free[sz].pop()))
                        _cached -= sz
        if not fits:
            return np.empty(shape, dt)
        try:
            from dosma_amd import _lib
            lib = _lib.load()
            out = ctypes.c_void_p()
            while drop:
                _apart.discard(drop[-1][1])
                lib.qmri_host_free(ctypes.c_void_p(drop[-1][1]))
                drop.pop()
            if lib.qmri_device_count() > 0 and lib.qmri_host_alloc(size, ctypes.byref(out)) == 0 and out.value:
                ptr = out.value
                if not _inherited(ptr, size):
                    _apart.add(ptr)
        except Exception:
            ptr = None
        if ptr is None:
            with _lock:
                _live -= size  # the reservation is rolled back; blocks that were not freed go back on the free list
                for sz, p in drop:
                    _free.setdefault(sz, []).append(p)
                    _cached += sz
            return np.empty(shape, dt)
    with _lock:
        _held[ptr] = size
    buf = (ctypes.c_ubyte * size).from_address(ptr)
    fin = weakref.finalize(buf, _release, ptr, size)
    fin.atexit = False  # nothing to recycle at interpreter exit (and no HIP call from an exit handler or a forked child)
    return np.frombuffer(buf, dtype=dt, count=count).reshape(shape)


def trim():
    """Return every cached block to the system (tests, long-running services between jobs)."""
    global _cached
    with _lock:
        old = dict(_free)
        _free.clear()
        _cached = 0
    blocks = [(p, s) for s, lst in old.items() for p in lst]
    if blocks:
        from dosma_amd import _lib
        lib = _lib.load()
        for p, _ in blocks:
            _apart.discard(p)
            lib.qmri_host_free(ctypes.c_void_p(p))


def cached_bytes():
    return _cached


def live_bytes():
    """Page-locked bytes currently owned by results that are still alive."""
    return _live


@atexit.register
def _shutdown():
    global _closed
    _closed = True
