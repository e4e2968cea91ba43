"""Python binding of libtsac_cuda.so (the C ABI declared in include/tsac_cuda.h).

Mirrors the reference's public analyzer API (include/tsac/audio_analyzer.hpp):
`CudaAnalyzer(package).encode(pcm, EncodeOptions) -> bytes` and
`.decode(stream) -> PcmAudio`, with tsac::Error surfacing as `TsacError`.
There is no CPU fallback: loading fails loudly if the library is missing, and
every GPU entry point fails with TSAC_CUDA_ERROR_DEVICE without a device.
"""
from __future__ import annotations

import ctypes
import dataclasses
import os
import pathlib
import shutil
import threading
import weakref

import numpy as np

HERE = pathlib.Path(__file__).resolve().parent
LIBRARY = HERE / "libtsac_cuda.so"
# Pack ID of every seeded package this library writes (16 lowercase hex digits,
# as the reference packer requires, src/weights/pack_main.cpp:748-751).
SEEDED_PACK_ID = "b200b200b200b200"

OK, ERROR, ERROR_DEVICE, ERROR_NUMERIC = 0, 1, 2, 3


class TsacError(RuntimeError):
    """tsac::Error equivalent; `.status` holds the C-ABI status code."""

    def __init__(self, message: str, status: int = ERROR):
        super().__init__(message)
        self.status = status


_lib = None
_lock = threading.Lock()


def library() -> ctypes.CDLL:
    global _lib
    with _lock:
        if _lib is None:
            if not LIBRARY.exists():
                raise TsacError(
                    f"{LIBRARY} is missing; build it with `make -C {HERE}` "
                    "(there is no CPU fallback)", ERROR_DEVICE)
            lib = ctypes.CDLL(str(LIBRARY))
            lib.tsac_cuda_last_error.restype = ctypes.c_char_p
            _lib = lib
        return _lib


def check(status: int) -> None:
    if status != OK:
        message = library().tsac_cuda_last_error().decode("utf-8", "replace")
        raise TsacError(message, status)


# ---------------------------------------------------------------- packages --
def write_seeded_sources(directory: os.PathLike, seed: int) -> None:
    check(library().tsac_cuda_write_seeded_sources(
        str(directory).encode(), ctypes.c_uint64(seed)))


def pack_models(source: os.PathLike, output: os.PathLike, pack_id: str = SEEDED_PACK_ID,
                include_transformer: bool = True) -> None:
    check(library().tsac_cuda_pack_models(
        str(source).encode(), str(output).encode(), pack_id.encode(),
        1 if include_transformer else 0))


def cache_root() -> pathlib.Path:
    root = os.environ.get("TSAC_B200_CACHE")
    return pathlib.Path(root) if root else pathlib.Path("/tmp/tsac_b200_models")


def seeded_package(seed: int = 0) -> pathlib.Path:
    """Directory of the seeded 20-file package (generated once, then cached).

    Safe under concurrent callers (one process per GPU on a fresh host): an
    exclusive lock on a file beside the cache serialises generation, the
    package is published by renaming a finished directory, and a process that
    waited finds it done."""
    import fcntl

    base = cache_root() / f"seed{seed}"
    package = base / "package"
    marker = package / "weights-manifest.cmake"
    if marker.exists():
        return package
    base.mkdir(parents=True, exist_ok=True)
    with open(base / "generate.lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)  # released when the file closes, or the process ends
        if marker.exists():
            return package
        source = base / "source"
        tmp = base / f"package.tmp{os.getpid()}"
        if tmp.exists():
            shutil.rmtree(tmp)
        if package.exists():  # left by an interrupted earlier attempt
            shutil.rmtree(package)
        write_seeded_sources(source, seed)
        pack_models(source, tmp)
        tmp.rename(package)
    return package


# ------------------------------------------------------------ kernel calls --
# Thin wrappers over the per-kernel C-ABI entry points.  Arguments are torch
# CUDA tensors (torch supplies device memory and streams; the arithmetic is
# entirely in this library's kernels).
def _dev(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def qlinear_scratch_bytes(m: int, k: int) -> int:
    lib = library()
    lib.tsac_cuda_qlinear_scratch_bytes.restype = ctypes.c_size_t
    return lib.tsac_cuda_qlinear_scratch_bytes(ctypes.c_size_t(m), ctypes.c_size_t(k))


def qlinear(weights, scales, bias, x, y, scratch, residual=None, error_word=None):
    """y[m][n] = bf16(W x + b) (+residual), all tensors on the device."""
    n, k = weights.shape
    m = x.shape[0]
    check(library().tsac_cuda_qlinear(
        _dev(weights), _dev(scales), _dev(bias), ctypes.c_size_t(k), ctypes.c_size_t(n), _dev(x),
        ctypes.c_size_t(m), _dev(residual), _dev(y), _dev(scratch),
        ctypes.c_size_t(scratch.numel() * scratch.element_size()), _dev(error_word), _stream()))


# ------------------------------------------------------- drafted decoding --
# Paged key/value cache, tree attention and draft verification
# (include/tsac_cuda.h states each operation).  Arguments are torch CUDA
# tensors; calls are asynchronous on the current stream of the tensors' device
# and may be captured into a CUDA graph.  Attention takes its temporary device
# memory from torch's allocator in each call, so that overlapping calls and
# graphs share none; reserve and compact, which must not overlap on one cache,
# keep theirs with it.
# There is no backward: tensors that require a gradient are refused outside
# torch.no_grad().
MAX_NODES = 64


class _PagedCacheStruct(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("pool", "tables", "counts", "lengths", "refs")] + \
               [(n, ctypes.c_size_t) for n in ("layers", "pages", "page_size", "kv_heads", "head_dim",
                                               "sequences", "max_pages")] + [("type", ctypes.c_int)]


_p, _n, _i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int
_DRAFTING = {
    "tsac_cuda_cache_reserve_scratch_bytes": (_n, [_n, _n]),
    "tsac_cuda_cache_reserve": (_i, [_p, _p, _p, _n, _n, _p, _n, _p, _p]),
    "tsac_cuda_cache_fork": (_i, [_p, _p, _p, _n, _p, _p]),
    "tsac_cuda_cache_release": (_i, [_p, _p, _p, _n, _p, _p]),
    "tsac_cuda_cache_append": (_i, [_p, _n, _p, _p, _p, _p, _p, _p, _p, _n, _n, _p, _p]),
    "tsac_cuda_cache_keep": (_i, [_p, _p, _p, _p, _p, _p, _n, _n, _p, _p]),
    "tsac_cuda_cache_compact_scratch_bytes": (_n, [_n]),
    "tsac_cuda_cache_compact": (_i, [_p, _p, _p, _p, _p, _n, _p, _p]),
    "tsac_cuda_tree_attention_scratch_bytes": (_n, [_p, _n, _n]),
    "tsac_cuda_tree_attention": (_i, [_p, _n, _p, _p, _p, _p, _p, _p, _p, _p, _n, _n, _n, ctypes.c_float,
                                      _p, _n, _p, _p]),
    "tsac_cuda_draft_verify": (_i, [_p, _p, _p, _p, _i, _p, _p, _p, _p, _p, _n, _n, _n, _p, _p, _p, _p, _p]),
}
_drafting_lib = None


def _drafting():
    """The library with the argument types of the drafting calls declared, once."""
    global _drafting_lib
    if _drafting_lib is None:
        lib = library()
        for name, (restype, argtypes) in _DRAFTING.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = restype, argtypes
        _drafting_lib = lib
    return _drafting_lib


class _Device:
    """Makes a tensor's device current for a call, and gives its current stream."""

    _known = {}

    def __init__(self, index):
        import torch
        self.index, self._cuda = index, torch.cuda
        # torch's direct queries where it has them: a call asks both, and is itself a few microseconds.
        self._current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        self._stream = (getattr(torch._C, "_cuda_getCurrentRawStream", None)
                        or (lambda i: torch.cuda.current_stream(i).cuda_stream))

    @classmethod
    def of(cls, index):
        on = cls._known.get(index)
        if on is None:
            on = cls._known[index] = cls(index)
        return on

    def stream(self) -> int:
        return self._stream(self.index)

    def ask(self, fn, *arguments) -> int:
        """What fn answers with the device current."""
        with self._cuda.device(self.index):
            return fn(*arguments)

    def call(self, fn, *arguments) -> None:
        if self._current() == self.index:
            status = fn(*arguments)
        else:
            status = self.ask(fn, *arguments)
        if status != OK:
            check(status)


def _whole(t, name, dtype, index, shape=None):
    """Address of a contiguous tensor of the given kind on device `index`; None gives a null pointer."""
    if t is None:
        return None
    if t.dtype is dtype and t.get_device() == index and t.is_contiguous() and (shape is None or t.shape == shape):
        return t.data_ptr()
    raise TsacError(f"{name} must be a contiguous {dtype} tensor on cuda:{index}"
                    + (f" of shape {tuple(shape)}" if shape is not None else ""))


def _error_word(word, index):
    if word is None:
        return None
    if word.numel() < 1 or word.element_size() != 4:
        raise TsacError("error_word must hold a 32-bit word")
    return _whole(word, "error_word", word.dtype, index)


_stride_arrays = {}


def _strides(values):
    """A C array of strides, kept for the next call with the same ones."""
    array = _stride_arrays.get(values)
    if array is None:
        if len(_stride_arrays) >= 1024:
            _stride_arrays.clear()
        array = _stride_arrays[values] = (ctypes.c_ssize_t * len(values))(*values)
    return array


def _no_gradient(t, name):
    """These calls have no backward: a gradient that autograd would have to carry through one is refused."""
    if t.requires_grad:
        import torch
        if torch.is_grad_enabled():
            raise TsacError(f"{name} requires a gradient, which the drafting calls do not carry: call them under torch.no_grad()")


def _rows(t, name, dtype, index, shape, found=None):
    """Address and strides of a [entry][node][head][dim] tensor with a contiguous last dimension; found: its shape, where known."""
    strides = t.stride()
    if t.dtype is not dtype or t.get_device() != index or (found or t.shape) != shape or (strides[-1] != 1 and shape[-1] > 1):
        raise TsacError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on cuda:{index}, its last dimension contiguous")
    if t.requires_grad:
        _no_gradient(t, name)
    array = _stride_arrays.get((strides, shape))
    if array is None:
        if len(_stride_arrays) >= 1024:
            _stride_arrays.clear()
        # A dimension of size one is never stepped over: its stride says nothing.
        array = _stride_arrays[strides, shape] = (ctypes.c_ssize_t * 3)(*[0 if n == 1 else s for n, s in zip(shape[:3], strides)])
    return t.data_ptr(), array


class PagedCache:
    """Token sequences over one pool of key/value pages (tsac_cuda_paged_cache).

    pool: [layers][2: keys, values][pages][page_size][kv_heads][head_dim], bf16
    or fp16; tables int32 [sequences][max_pages]; counts, lengths int32
    [sequences]; refs int32 [pages].  The tensors stay the caller's: reading,
    saving or replacing their contents between calls is fine.  The tensors
    themselves stay the same ones: their addresses are bound here, and a cache
    over other tensors is a new object.  Keep the object as long as a CUDA graph
    that was captured from its calls.
    """

    _bound = frozenset(("pool", "tables", "counts", "lengths", "refs"))

    def __setattr__(self, name, value):
        # (Not by __dict__: asking for it would make every later attribute of the object slower.)
        if name in self._bound and getattr(self, name, value) is not value:
            raise TsacError(f"{name} is bound to the cache: copy into it, or make a PagedCache over other tensors")
        object.__setattr__(self, name, value)

    def __init__(self, pool, tables, counts, lengths, refs):
        import torch
        if pool.dim() != 6 or pool.shape[1] != 2 or not pool.is_cuda or pool.dtype not in (torch.bfloat16, torch.float16):
            raise TsacError("pool must be a bf16 or fp16 CUDA tensor [layers][2][pages][page_size][kv_heads][head_dim]")
        _no_gradient(pool, "pool")
        self.pool, self.tables, self.counts, self.lengths, self.refs = pool, tables, counts, lengths, refs
        self.device, self.index, self.dtype = pool.device, pool.get_device(), pool.dtype
        self._torch, self._int, self._bytes = torch, torch.int32, torch.empty(0, dtype=torch.uint8, device=self.device)
        if tables.dim() != 2:
            raise TsacError("tables must be [sequences][max_pages]")
        self.layers, _, self.pages, self.page_size, self.kv_heads, self.head_dim = pool.shape
        self.sequences, self.max_pages = tables.shape
        s = _PagedCacheStruct()
        s.pool = _whole(pool, "pool", pool.dtype, self.index)
        s.tables = _whole(tables, "tables", self._int, self.index)
        s.counts = _whole(counts, "counts", self._int, self.index, (self.sequences,))
        s.lengths = _whole(lengths, "lengths", self._int, self.index, (self.sequences,))
        s.refs = _whole(refs, "refs", self._int, self.index, (self.pages,))
        for name in ("layers", "pages", "page_size", "kv_heads", "head_dim", "sequences", "max_pages"):
            setattr(s, name, getattr(self, name))
        s.type = 0 if pool.dtype == torch.bfloat16 else 1
        self._struct, self._lib, self._on = s, _drafting(), _Device.of(self.index)
        self._cache = ctypes.addressof(s)
        self._scratches, self._attention_bytes = [], {}

    @classmethod
    def empty(cls, layers, pages, page_size, kv_heads, head_dim, sequences, max_pages, dtype=None, device="cuda"):
        """A cache whose sequences hold nothing."""
        import torch
        ints = dict(dtype=torch.int32, device=device)
        return cls(torch.zeros((layers, 2, pages, page_size, kv_heads, head_dim), dtype=dtype or torch.bfloat16, device=device),
                   torch.full((sequences, max_pages), -1, **ints), torch.zeros(sequences, **ints),
                   torch.zeros(sequences, **ints), torch.zeros(pages, **ints))

    def _list(self, sequences, count):
        return _whole(sequences, "sequences", self._int, self.index, (count,))

    def _word(self, error_word):
        return _error_word(error_word, self.index)

    def _temporary(self, nbytes):
        return self._bytes.new_empty(max(nbytes, 16))

    def _kept(self, nbytes):
        """Temporary memory of the calls that change the cache, which must not overlap: kept from one to the next.
        A larger one is added, not exchanged: a captured graph goes on using the one that it was captured with."""
        stream = self._on.stream()
        if not self._scratches or self._scratches[-1][0].numel() < nbytes:
            last = self._scratches[-1][0].numel() if self._scratches else 0
            self._scratches.append((self._temporary(max(nbytes, 2 * last)), stream))
        scratch, owner = self._scratches[-1]
        if owner != stream:  # the allocator must not hand it out again before this stream is done with it
            scratch.record_stream(self._torch.cuda.current_stream(self.index))
        return scratch

    def reserve(self, positions, sequences=None, slots=None, error_word=None):
        """Makes positions[i] further positions of each sequence writable (all or nothing)."""
        if positions.dim() != 1:
            raise TsacError("positions must be [entry]")
        count = positions.shape[0]
        slots = slots or self.max_pages
        nbytes = self._lib.tsac_cuda_cache_reserve_scratch_bytes(count, slots)
        scratch = self._kept(nbytes)
        self._on.call(self._lib.tsac_cuda_cache_reserve, self._cache, self._list(sequences, count),
                      _whole(positions, "positions", self._int, self.index, (count,)), count, slots,
                      scratch.data_ptr(), nbytes, self._word(error_word), self._on.stream())

    def fork(self, parents, children, error_word=None):
        """children[i], empty so far, shares the committed pages of parents[i]."""
        if parents.dim() != 1:
            raise TsacError("parents must be [entry]")
        count = parents.shape[0]
        self._on.call(self._lib.tsac_cuda_cache_fork, self._cache,
                      _whole(parents, "parents", self._int, self.index, (count,)),
                      _whole(children, "children", self._int, self.index, (count,)), count,
                      self._word(error_word), self._on.stream())

    def release(self, sequences=None, positions=None, error_word=None):
        """Gives back the pages behind positions[i] (None: all) of each sequence."""
        if sequences is not None and sequences.dim() != 1:
            raise TsacError("sequences must be [entry]")
        count = sequences.shape[0] if sequences is not None else self.sequences
        self._on.call(self._lib.tsac_cuda_cache_release, self._cache, self._list(sequences, count),
                      _whole(positions, "positions", self._int, self.index, (count,)), count,
                      self._word(error_word), self._on.stream())

    def append(self, layer, keys, values, nodes=None, sequences=None, starts=None, error_word=None):
        """Stores [entry][node][kv_heads][head_dim] rows of one layer behind each sequence's length (or at starts)."""
        found = keys.shape
        if len(found) != 4:
            raise TsacError("keys must be [entry][node][kv_heads][head_dim]")
        count, most, _, _ = found
        shape, index, ints = (count, most, self.kv_heads, self.head_dim), self.index, self._int
        k, key_strides = _rows(keys, "keys", self.dtype, index, shape, found)
        v, value_strides = _rows(values, "values", self.dtype, index, shape)
        self._on.call(self._lib.tsac_cuda_cache_append, self._cache, layer, k, key_strides, v, value_strides,
                      sequences if sequences is None else _whole(sequences, "sequences", ints, index, (count,)),
                      nodes if nodes is None else _whole(nodes, "nodes", ints, index, (count,)),
                      starts if starts is None else _whole(starts, "starts", ints, index, (count,)), count, most,
                      error_word if error_word is None else self._word(error_word), self._on.stream())

    def keep(self, path, accepted, starts=None, lengths_out=None, sequences=None, error_word=None):
        """Keeps rows start + path[i][:accepted[i]], in every layer, as the next positions."""
        if path.dim() != 2:
            raise TsacError("path must be [entry][width]")
        count, width = path.shape
        out = self.lengths if lengths_out is None else lengths_out
        self._on.call(self._lib.tsac_cuda_cache_keep, self._cache, self._list(sequences, count),
                      _whole(path, "path", self._int, self.index),
                      _whole(accepted, "accepted", self._int, self.index, (count,)),
                      _whole(starts, "starts", self._int, self.index, (count,)),
                      _whole(out, "lengths_out", self._int, self.index, (self.sequences,)), count, width,
                      self._word(error_word), self._on.stream())

    def compact(self, tables_out=None, refs_out=None, live=None, error_word=None):
        """Moves the pages in use to the lower end of the pool; returns their number (device int32 [1])."""
        live = self._torch.empty(1, dtype=self._int, device=self.device) if live is None else live
        scratch = self._kept(self._lib.tsac_cuda_cache_compact_scratch_bytes(self.pages))
        self._on.call(self._lib.tsac_cuda_cache_compact, self._cache,
                      _whole(self.tables if tables_out is None else tables_out, "tables_out", self._int, self.index,
                             self.tables.shape),
                      _whole(self.refs if refs_out is None else refs_out, "refs_out", self._int, self.index, (self.pages,)),
                      _whole(live, "live", self._int, self.index, (1,)), scratch.data_ptr(), scratch.numel(),
                      self._word(error_word), self._on.stream())
        return live

    def attention(self, layer, query, parents, out=None, nodes=None, sequences=None, scale=None, lse=None,
                  error_word=None):
        """Attention of each tree's nodes over the cache: query [entry][node][heads][head_dim] -> out."""
        found = query.shape
        if len(found) != 4:
            raise TsacError("query must be [entry][node][heads][head_dim]")
        count, most, heads, _ = found
        shape, index, ints, on = (count, most, heads, self.head_dim), self.index, self._int, self._on
        out = query.new_empty(shape) if out is None else out
        q, query_strides = _rows(query, "query", self.dtype, index, shape, found)
        o, out_strides = _rows(out, "out", self.dtype, index, shape)
        nbytes = self._attention_bytes.get((heads, most))
        if nbytes is None:
            # By the cache's device: the size depends on its multiprocessors.
            nbytes = on.ask(self._lib.tsac_cuda_tree_attention_scratch_bytes, self._cache, heads, most)
            self._attention_bytes[heads, most] = nbytes
        scratch = self._temporary(nbytes)
        on.call(self._lib.tsac_cuda_tree_attention, self._cache, layer,
                None if sequences is None else _whole(sequences, "sequences", ints, index, (count,)),
                _whole(parents, "parents", ints, index, (count, most)),
                None if nodes is None else _whole(nodes, "nodes", ints, index, (count,)), q, query_strides, o, out_strides,
                None if lse is None else _whole(lse, "lse", self._torch.float32, index, (count, most, heads)), heads, count,
                most, self.head_dim ** -0.5 if scale is None else scale, scratch.data_ptr(), nbytes,
                None if error_word is None else _error_word(error_word, index), on.stream())
        return out


_verify_types = {}


def draft_verify(target, tokens, parents, coins, draws, draft=None, nodes=None, out=None, error_word=None):
    """Checks trees of drafted tokens against the target's probabilities (tsac_cuda_draft_verify).

    target [batch][nodes][vocab] (draft the same, or None), tokens and parents
    int32 [batch][nodes], coins f32 [batch][nodes], draws f32 [batch] in [0, 1).
    Returns (accepted [batch], path [batch][nodes], token [batch]), int32, in
    `out` when given."""
    lib = _drafting()
    if not _verify_types:
        import torch
        _verify_types.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, "ints": torch.int32})
    if target.dim() != 3 or not target.is_cuda:
        raise TsacError("target must be a CUDA tensor [batch][nodes][vocab]")
    shape = target.shape
    batch, most, vocab = shape
    index, kind, ints, floats = target.get_device(), target.dtype, _verify_types["ints"], draws.dtype
    strides = target.stride()
    if kind not in _verify_types or (strides[2] != 1 and vocab > 1):
        raise TsacError("target must be bf16, fp16 or fp32 [batch][nodes][vocab], the vocabulary contiguous")
    if draft is not None and (draft.dtype is not kind or draft.get_device() != index or draft.shape != shape
                              or (draft.stride(2) != 1 and vocab > 1)):
        raise TsacError("draft must be of the target's type and shape, the vocabulary contiguous")
    if _verify_types.get(floats) != 2:
        raise TsacError("draws must be float32")
    rows, ones = (batch, most), (batch,)
    q, q_strides = (None, None) if draft is None else (draft.data_ptr(), _strides(draft.stride()[:2]))
    tokens_at, parents_at = _whole(tokens, "tokens", ints, index, rows), _whole(parents, "parents", ints, index, rows)
    if out is None:
        accepted, path, token = tokens.new_empty(batch), tokens.new_empty(rows), tokens.new_empty(batch)
        places = accepted.data_ptr(), path.data_ptr(), token.data_ptr()
    else:
        accepted, path, token = out
        places = (_whole(accepted, "accepted", ints, index, ones), _whole(path, "path", ints, index, rows),
                  _whole(token, "token", ints, index, ones))
    on = _Device.of(index)
    on.call(lib.tsac_cuda_draft_verify, target.data_ptr(), _strides(strides[:2]), q, q_strides, _verify_types[kind],
            tokens_at, parents_at, _whole(coins, "coins", floats, index, rows), _whole(draws, "draws", floats, index, ones),
            None if nodes is None else _whole(nodes, "nodes", ints, index, ones), batch, most, vocab, *places,
            None if error_word is None else _error_word(error_word, index), on.stream())
    return accepted, path, token


# --------------------------------------------------------------- analyzer --
@dataclasses.dataclass
class EncodeOptions:
    """tsac::EncodeOptions (include/tsac/audio_analyzer.hpp:16-22)."""
    method: str = "normal"          # "normal" or "fast"
    codebooks: int = 0              # 0: model maximum
    separate_channels: bool = False
    entropy_batch: int | None = None  # None: automatic


class _Options(ctypes.Structure):
    _fields_ = [("method", ctypes.c_int), ("codebooks", ctypes.c_uint),
                ("separate_channels", ctypes.c_int), ("entropy_batch", ctypes.c_int)]


def _options(o: EncodeOptions | None) -> _Options:
    o = o or EncodeOptions()
    if o.method not in ("normal", "fast"):
        raise TsacError("invalid coding method")
    return _Options(1 if o.method == "normal" else 0, o.codebooks,
                    1 if o.separate_channels else 0, o.entropy_batch or 0)


@dataclasses.dataclass
class PcmAudio:
    """tsac::PcmAudio: interleaved float32 samples [frames][channels]."""
    samples: np.ndarray
    channels: int


def _adopt(ptr, count, dtype):
    """A numpy view of a library-allocated buffer that frees it (tsac_cuda_free)
    when the last array using it is collected: large results (decoded PCM) are
    not copied a second time."""
    lib = library()
    if not count:
        lib.tsac_cuda_free(ptr)
        return np.zeros(0, dtype)
    address = ptr.value if isinstance(ptr, ctypes.c_void_p) else int(ptr)
    storage = (np.ctypeslib.as_ctypes_type(dtype) * count).from_address(address)
    weakref.finalize(storage, lib.tsac_cuda_free, ctypes.c_void_p(address))
    return np.frombuffer(storage, dtype)


def _take(ptr, count, dtype):
    """Copy a library-allocated buffer into numpy and free it."""
    lib = library()
    if count:
        arr = np.ctypeslib.as_array(ctypes.cast(ptr, ctypes.POINTER(np.ctypeslib.as_ctypes_type(dtype))),
                                    shape=(count,)).copy()
    else:
        arr = np.zeros(0, dtype)
    lib.tsac_cuda_free(ptr)
    return arr


class CudaAnalyzer:
    """B200 implementation of tsac::AudioAnalyzer (include/tsac/audio_analyzer.hpp:30-37).

    Calls are synchronous; one instance is used by one thread at a time.
    """

    def __init__(self, package: os.PathLike, device: int = 0):
        lib = library()
        self._ctx = ctypes.c_void_p()
        check(lib.tsac_cuda_context_create(str(package).encode(), device, ctypes.byref(self._ctx)))

    def set_exact_synthesis(self, exact: bool) -> None:
        """Exact (bit-identical PCM) or tensor-core (within tolerance) synthesis."""
        check(library().tsac_cuda_set_exact_synthesis(self._ctx, 1 if exact else 0))

    def set_host_threads(self, threads: int) -> None:
        """Host range-coding worker budget (0: automatic, at most 256), the
        thread count AppleArmAnalyzer takes (src/apple-arm/audio_analyzer.cpp:93)."""
        if threads < 0:
            raise TsacError("invalid thread count")
        check(library().tsac_cuda_set_host_threads(self._ctx, ctypes.c_uint(threads)))

    def set_fast_analysis(self, margin: float) -> None:
        """Certified fast analysis: 0 = exact analysis; margin > 0 = fused
        multiply-add analysis with every frame whose RVQ decision lead is below
        `margin` recomputed exactly (streams stay the reference's)."""
        check(library().tsac_cuda_set_fast_analysis(self._ctx, ctypes.c_float(margin)))

    def fast_analysis_stats(self):
        """(central frames coded, frames flagged uncertain, frames recomputed exactly)."""
        f, u, r = ctypes.c_uint64(), ctypes.c_uint64(), ctypes.c_uint64()
        check(library().tsac_cuda_fast_analysis_stats(self._ctx, ctypes.byref(f), ctypes.byref(u),
                                                      ctypes.byref(r)))
        return f.value, u.value, r.value

    def close(self):
        if self._ctx:
            library().tsac_cuda_context_destroy(self._ctx)
            self._ctx = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def encode(self, pcm: np.ndarray, options: EncodeOptions | None = None,
               with_bits: bool = False):
        """pcm: float32 [samples][channels] (interleaved) or any 2-D strided view."""
        pcm = np.asarray(pcm, dtype=np.float32)
        if pcm.ndim == 1:
            pcm = pcm[:, None]
        samples, channels = pcm.shape
        out = ctypes.c_void_p()
        nbytes, bits = ctypes.c_size_t(), ctypes.c_size_t()
        opts = _options(options)
        check(library().tsac_cuda_encode(
            self._ctx, pcm.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(channels),
            ctypes.c_size_t(samples), ctypes.c_ssize_t(pcm.strides[1] // 4),
            ctypes.c_ssize_t(pcm.strides[0] // 4), ctypes.byref(opts), ctypes.byref(out),
            ctypes.byref(nbytes), ctypes.byref(bits)))
        data = _take(out, nbytes.value, np.uint8).tobytes()
        return (data, bits.value) if with_bits else data

    def encode_symbol_bits(self, pcm: np.ndarray, options: EncodeOptions | None = None):
        """encode() plus each symbol's bits in entropy order (what an
        EntropyObserver's after_symbol receives); an empty array for fast streams."""
        pcm = np.asarray(pcm, dtype=np.float32)
        if pcm.ndim == 1:
            pcm = pcm[:, None]
        samples, channels = pcm.shape
        out, per_symbol = ctypes.c_void_p(), ctypes.c_void_p()
        nbytes, count = ctypes.c_size_t(), ctypes.c_size_t()
        opts = _options(options)
        check(library().tsac_cuda_encode_symbol_bits(
            self._ctx, pcm.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(channels),
            ctypes.c_size_t(samples), ctypes.c_ssize_t(pcm.strides[1] // 4),
            ctypes.c_ssize_t(pcm.strides[0] // 4), ctypes.byref(opts), ctypes.byref(out),
            ctypes.byref(nbytes), ctypes.byref(per_symbol), ctypes.byref(count)))
        data = _take(out, nbytes.value, np.uint8).tobytes()
        return data, _take(per_symbol, count.value, np.uint32)

    def decode(self, stream: bytes) -> PcmAudio:
        out = ctypes.c_void_p()
        samples, channels = ctypes.c_size_t(), ctypes.c_uint()
        check(library().tsac_cuda_decode(self._ctx, stream, ctypes.c_size_t(len(stream)),
                                         ctypes.byref(out), ctypes.byref(samples),
                                         ctypes.byref(channels)))
        data = _adopt(out, samples.value, np.float32)
        return PcmAudio(data.reshape(-1, channels.value), channels.value)

    def encode_batch(self, pcms, options: EncodeOptions | None = None):
        pcms = [np.ascontiguousarray(p, dtype=np.float32).reshape(p.shape[0], -1) for p in pcms]
        n = len(pcms)
        ptrs = (ctypes.c_void_p * n)(*[p.ctypes.data for p in pcms])
        chans = (ctypes.c_size_t * n)(*[p.shape[1] for p in pcms])
        sams = (ctypes.c_size_t * n)(*[p.shape[0] for p in pcms])
        outs = (ctypes.c_void_p * n)()
        sizes = (ctypes.c_size_t * n)()
        opts = _options(options)
        check(library().tsac_cuda_encode_batch(self._ctx, ctypes.c_size_t(n), ptrs, chans, sams,
                                               ctypes.byref(opts), outs, sizes))
        return [_take(ctypes.c_void_p(outs[i]), sizes[i], np.uint8).tobytes() for i in range(n)]

    def decode_batch(self, streams):
        n = len(streams)
        bufs = [ctypes.create_string_buffer(s, len(s)) for s in streams]
        ptrs = (ctypes.c_void_p * n)(*[ctypes.addressof(b) for b in bufs])
        sizes = (ctypes.c_size_t * n)(*[len(s) for s in streams])
        outs = (ctypes.c_void_p * n)()
        samples = (ctypes.c_size_t * n)()
        chans = (ctypes.c_uint * n)()
        check(library().tsac_cuda_decode_batch(self._ctx, ctypes.c_size_t(n), ptrs, sizes, outs,
                                               samples, chans))
        return [PcmAudio(_adopt(ctypes.c_void_p(outs[i]), samples[i], np.float32)
                         .reshape(-1, chans[i]), chans[i]) for i in range(n)]

    # ---- pipeline stages (parity tests) ---------------------------------
    def analyze_tokens(self, pcm: np.ndarray, options: EncodeOptions | None = None):
        pcm = np.ascontiguousarray(pcm, dtype=np.float32).reshape(pcm.shape[0], -1)
        out = ctypes.c_void_p()
        count = ctypes.c_size_t()
        opts = _options(options)
        check(library().tsac_cuda_analyze_tokens(
            self._ctx, pcm.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(pcm.shape[1]),
            ctypes.c_size_t(pcm.shape[0]), ctypes.byref(opts), ctypes.byref(out),
            ctypes.byref(count)))
        return _take(out, count.value, np.uint16)

    def dac_analysis(self, channels: int, pcm: np.ndarray) -> np.ndarray:
        pcm = np.ascontiguousarray(pcm, dtype=np.float32)
        frames = pcm.size // channels
        latent = np.zeros((frames // 512, 1024), np.float32)
        check(library().tsac_cuda_dac_analysis(self._ctx, channels, pcm.ctypes.data_as(ctypes.c_void_p),
                                                ctypes.c_size_t(frames),
                                                latent.ctypes.data_as(ctypes.c_void_p)))
        return latent

    def dac_synthesis(self, channels: int, latent: np.ndarray) -> np.ndarray:
        latent = np.ascontiguousarray(latent, dtype=np.float32)
        frames = latent.size // 1024
        pcm = np.zeros((frames * 512, channels), np.float32)
        check(library().tsac_cuda_dac_synthesis(self._ctx, channels,
                                                 latent.ctypes.data_as(ctypes.c_void_p),
                                                 ctypes.c_size_t(frames),
                                                 pcm.ctypes.data_as(ctypes.c_void_p)))
        return pcm

    def rvq_encode(self, channels: int, books: int, latent: np.ndarray) -> np.ndarray:
        latent = np.ascontiguousarray(latent, dtype=np.float32)
        frames = latent.size // 1024
        tokens = np.zeros((frames, books), np.uint16)
        check(library().tsac_cuda_rvq_encode(self._ctx, channels, books,
                                             latent.ctypes.data_as(ctypes.c_void_p),
                                             ctypes.c_size_t(frames),
                                             tokens.ctypes.data_as(ctypes.c_void_p)))
        return tokens

    def rvq_decode(self, channels: int, books: int, tokens: np.ndarray) -> np.ndarray:
        tokens = np.ascontiguousarray(tokens, dtype=np.uint16)
        frames = tokens.size // books
        latent = np.zeros((frames, 1024), np.float32)
        check(library().tsac_cuda_rvq_decode(self._ctx, channels, books,
                                             tokens.ctypes.data_as(ctypes.c_void_p),
                                             ctypes.c_size_t(frames),
                                             latent.ctypes.data_as(ctypes.c_void_p)))
        return latent

    def transformer_probabilities(self, channels, groups, books, frames, batch, tokens,
                                  probabilities=True):
        tokens = np.ascontiguousarray(tokens, dtype=np.uint16)
        symbols = frames * groups * books
        probs = np.zeros((symbols, 1024), np.float32) if probabilities else None
        q15 = np.zeros((symbols, 10), np.uint16)
        check(library().tsac_cuda_transformer_probabilities(
            self._ctx, channels, groups, books, ctypes.c_size_t(frames), batch,
            tokens.ctypes.data_as(ctypes.c_void_p),
            probs.ctypes.data_as(ctypes.c_void_p) if probs is not None else None,
            q15.ctypes.data_as(ctypes.c_void_p)))
        return probs, q15

    def pack_normal(self, channels, groups, books, frames, batch, tokens) -> bytes:
        tokens = np.ascontiguousarray(tokens, dtype=np.uint16)
        out = ctypes.c_void_p()
        nbytes = ctypes.c_size_t()
        check(library().tsac_cuda_pack_normal(self._ctx, channels, groups, books,
                                              ctypes.c_size_t(frames), batch,
                                              tokens.ctypes.data_as(ctypes.c_void_p),
                                              ctypes.byref(out), ctypes.byref(nbytes)))
        return _take(out, nbytes.value, np.uint8).tobytes()


def stream_info(stream: bytes):
    """(channels, samples_per_channel, symbols) of a .tsac stream."""
    ch, spc, sym = ctypes.c_uint(), ctypes.c_size_t(), ctypes.c_size_t()
    check(library().tsac_cuda_stream_info(stream, ctypes.c_size_t(len(stream)), ctypes.byref(ch),
                                          ctypes.byref(spc), ctypes.byref(sym)))
    return ch.value, spc.value, sym.value


def unpack_fast(stream: bytes) -> np.ndarray:
    """Token indices of a fast-method stream (header and CRC checked)."""
    ptr, n = ctypes.POINTER(ctypes.c_uint16)(), ctypes.c_size_t()
    check(library().tsac_cuda_unpack_fast(stream, ctypes.c_size_t(len(stream)), ctypes.byref(ptr),
                                          ctypes.byref(n)))
    return _take(ptr, n.value, np.uint16)


def token_crc32(tokens) -> int:
    """CRC-32 (polynomial 0x04c11db7) of token indices, as a normal header stores it."""
    t = np.ascontiguousarray(tokens, dtype=np.uint16)
    fn = library().tsac_cuda_token_crc32
    fn.restype = ctypes.c_uint32
    return fn(t.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(t.size))


def encode_batch_device(analyzer: "CudaAnalyzer", pcm_tensors, options: EncodeOptions | None = None):
    """Encode HBM-resident interleaved PCM (torch CUDA float32 [samples][channels])."""
    n = len(pcm_tensors)
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in pcm_tensors])
    chans = (ctypes.c_size_t * n)(*[t.shape[1] for t in pcm_tensors])
    sams = (ctypes.c_size_t * n)(*[t.shape[0] for t in pcm_tensors])
    outs = (ctypes.c_void_p * n)()
    sizes = (ctypes.c_size_t * n)()
    opts = _options(options)
    check(library().tsac_cuda_encode_batch_device(analyzer._ctx, ctypes.c_size_t(n), ptrs, chans,
                                                  sams, ctypes.byref(opts), outs, sizes))
    return [_take(ctypes.c_void_p(outs[i]), sizes[i], np.uint8).tobytes() for i in range(n)]


def decode_batch_device(analyzer: "CudaAnalyzer", streams, out_tensors):
    """Decode into HBM-resident PCM tensors (torch CUDA float32, channels x samples each)."""
    n = len(streams)
    bufs = [ctypes.create_string_buffer(s, len(s)) for s in streams]
    ptrs = (ctypes.c_void_p * n)(*[ctypes.addressof(b) for b in bufs])
    sizes = (ctypes.c_size_t * n)(*[len(s) for s in streams])
    outs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in out_tensors])
    check(library().tsac_cuda_decode_batch_device(analyzer._ctx, ctypes.c_size_t(n), ptrs, sizes,
                                                  outs))
