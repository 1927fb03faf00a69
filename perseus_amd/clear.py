"""The clear side of an encrypted transformer block, on the device: rotary positions, the norms of queries and keys with
the rotation in the same pass, and attention over packed prompts, chunks and single tokens, over keys packed, in caches or in
pages; the weight that cached keys gather, and the eviction of those of least weight.

The encrypted scoring (perseus_amd.attention) multiplies plaintext queries into an encrypted cache of keys. `Clear` makes
those queries and keys from projected rows, and the attention in the clear that the decrypted scores are held against: its
log-sum-exp turns a score into a probability, exp(score - lse). That cache holds a fixed number of keys: `key_weights` sums
those probabilities for each key, `evict` and `move_rows` cut a longer cache to the keys that gathered most
(attention.PagedBlock uses them all). The kernels are csrc/rotary.hip, csrc/attend.h (attend.hip, attend_paged.hip),
csrc/weigh.hip and csrc/evict.hip behind the pcx entries of the same names (include/pc_hip.h), which a C caller uses directly.

Tensors are `Array`s (a DevBuf with a shape and a type) or any device tensor of another library with data_ptr(), shape,
stride() and dtype; their last dimension is dense, the others may have any stride the entry takes. Everything is enqueued
on the Clear's stream; nothing is allocated, synchronised or copied by a call.
"""
import ctypes as C
import struct

import numpy as np

from ._lib import LIB, check
from .engine import DevBuf

TYPES = {"bf16": 0, "f16": 1, "f32": 2}
SIZES = {"bf16": 2, "f16": 2, "f32": 4, "i32": 4, "i64": 8}
_NAMES = {"bfloat16": "bf16", "float16": "f16", "half": "f16", "float32": "f32", "int32": "i32", "int64": "i64"}
_known = {k: k for k in SIZES}


def _type(dtype):
    """the short name of a tensor's dtype ("bf16", torch.bfloat16, ...)"""
    name = _known.get(dtype)
    if name is None:
        name = _NAMES.get(str(dtype).rsplit(".", 1)[-1])
        if name is None:
            raise ValueError(f"type {dtype}: not one of {', '.join(SIZES)}")
        _known[dtype] = name
    return name


def to_bf16(a):
    """The bfloat16 words (uint16) nearest to float32 values, ties to even."""
    w = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((w + 0x7FFF + ((w >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(w.view(np.float32)), np.uint16(0x7FC0) | (w >> 16).astype(np.uint16), r)


def from_bf16(w):
    """The float32 values of bfloat16 words (uint16)."""
    return (np.ascontiguousarray(w, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Array:
    """A device tensor: a DevBuf (from word `offset` on), a shape, a type of SIZES, row-major unless strides (in elements)
    are given."""

    is_cuda = True

    def __init__(self, shape, dtype, buf=None, offset=0, strides=None):
        self.shape, self.dtype = tuple(int(x) for x in shape), _type(dtype)
        if strides is None:
            strides, n = [], 1
            for x in reversed(self.shape):
                strides.insert(0, n)
                n *= x
        self._strides = tuple(int(x) for x in strides)
        if len(self._strides) != len(self.shape) or min(self._strides, default=0) < 0:
            raise ValueError("one stride, not negative, for each dimension")
        last = 1 + sum((n - 1) * st for n, st in zip(self.shape, self._strides)) if all(self.shape) else 0
        self.buf = DevBuf(-(-last * SIZES[self.dtype] // 4)) if buf is None else buf
        self.offset = int(offset)
        if self.offset < 0 or 4 * self.offset + last * SIZES[self.dtype] > 4 * self.buf.words:
            raise ValueError("the tensor leaves its buffer")

    @classmethod
    def of(cls, a, dtype=None, stream=None):
        """A dense copy of host values: float arrays as f32 unless dtype says bf16 or f16, integers as i32 or, where that does
        not hold their type, i64."""
        a = np.asarray(a)
        if not dtype:
            whole = a.dtype.kind in "iu"
            dtype = "f32" if not whole else "i32" if np.can_cast(a.dtype, np.int32) else "i64"
        dtype = _type(dtype)
        kind = {"f16": np.float16, "f32": np.float32, "i32": np.int32, "i64": np.int64}
        raw = np.ascontiguousarray(to_bf16(a) if dtype == "bf16" else a.astype(kind[dtype])).tobytes()
        x = cls(a.shape, dtype)
        if raw:
            x.buf.upload(np.frombuffer(raw + bytes(-len(raw) % 4), np.uint32), stream)
        return x

    def numpy(self, stream=None):
        """The values on the host (bf16 and f16 as float32), after the work on `stream`."""
        kind = {"bf16": np.uint16, "f16": np.float16, "f32": np.float32, "i32": np.int32, "i64": np.int64}[self.dtype]
        if not all(self.shape):
            return np.zeros(self.shape, np.float32 if self.dtype in TYPES else kind)
        last = 1 + sum((n - 1) * st for n, st in zip(self.shape, self._strides))
        words = self.buf.download(stream=stream, offset=self.offset, words=-(-last * SIZES[self.dtype] // 4))
        flat = words.view(kind)
        a = np.lib.stride_tricks.as_strided(flat, self.shape, [st * flat.itemsize for st in self._strides])
        return from_bf16(a) if self.dtype == "bf16" else a.astype(np.float32) if self.dtype == "f16" else a.copy()

    def heads(self, first, count):
        """Heads first .. first + count - 1 of a tensor [tokens][heads][dim], over the same memory."""
        t, h, d = self.shape
        if not 0 <= first <= first + count <= h:
            raise ValueError("heads out of range")
        at = first * self._strides[1] * SIZES[self.dtype]
        if at % 4:
            raise ValueError("the first head does not begin at a whole word")
        return Array((t, count, d), self.dtype, self.buf, self.offset + at // 4, self._strides)

    def data_ptr(self):
        return self.buf.ptr.value + 4 * self.offset

    def stride(self):
        return self._strides

    def numel(self):
        return int(np.prod(self.shape, dtype=np.int64))

    def is_contiguous(self):
        n = 1
        for size, step in zip(reversed(self.shape), reversed(self._strides)):
            if size != 1 and step != n:
                return not all(self.shape)
            n *= size
        return True


# ---------------------------------------------------------------------------------------------------- rotation tables


def rotary_rates(rot, base=10000.0, scaling=None):
    """The angle per place of each of the rot / 2 pairs, base^(-2 i / rot), in 64 bits. scaling stretches them for contexts
    longer than the `original` places a model was trained on, by `factor`:
    ("linear", factor): every angle divided by factor;
    ("base", factor): the base times factor^(rot / (rot - 2)), so that the slowest pair is stretched by the factor and the
    fastest keeps its pace;
    ("by_turns", factor, original, low, high): pairs that turn fewer than `low` times in `original` places are divided by
    factor, those that turn more than `high` times kept, a linear ramp over the turns between."""
    if rot % 2 or rot < 2:
        raise ValueError("rot is even and at least 2")
    i = np.arange(0, rot, 2, dtype=np.float64)
    if scaling is None:
        return float(base) ** (-i / rot)
    kind, factor = scaling[0], float(scaling[1])
    if factor <= 0:
        raise ValueError("the factor is positive")
    if kind == "linear":
        return float(base) ** (-i / rot) / factor
    if kind == "base":
        if rot < 4:
            raise ValueError("a stretched base needs two pairs or more")
        return (float(base) * factor ** (rot / (rot - 2))) ** (-i / rot)
    if kind == "by_turns":
        original, low, high = (float(x) for x in scaling[2:])
        if not 0 < low < high:
            raise ValueError("low below high")
        rate = float(base) ** (-i / rot)
        keep = np.clip((original * rate / (2 * np.pi) - low) / (high - low), 0, 1)
        return rate * (keep + (1 - keep) / factor)
    raise ValueError(f"scaling {kind}: linear, base or by_turns")


def rotary_table(places, rot, base=10000.0, scaling=None, magnitude=1.0):
    """cos and sin of every place and pair, float32 [places][rot / 2][2], rounded once from 64-bit angles; magnitude scales
    both (long-context scalings that sharpen the scores rotate by a factor)."""
    angle = np.arange(places, dtype=np.float64)[:, None] * rotary_rates(rot, base, scaling)
    return (np.stack([np.cos(angle), np.sin(angle)], -1) * magnitude).astype(np.float32)


# ---------------------------------------------------------------------------------------------------- argument structs

_vp, _i32, _i64, _f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float


def _ref(name):
    return [(name, _vp), (name + "_token", _i64), (name + "_head", _i64)]


class RotaryArgs(C.Structure):
    """include/pc_hip.h RotaryArgs (each HeadsRef as its three fields)."""
    _fields_ = [*_ref("x"), *_ref("out"), ("positions", _vp), ("table", _vp), ("places", _i64), ("tokens", _i32),
                ("heads", _i32), ("dim", _i32), ("rot", _i32), ("type", _i32), ("interleaved", _i32), ("inverse", _i32),
                ("pad", _i32)]


class QkNormRotaryArgs(C.Structure):
    """include/pc_hip.h QkNormRotaryArgs."""
    _fields_ = [*_ref("q"), *_ref("k"), *_ref("v"), *_ref("q_out"), *_ref("k_out"), *_ref("v_out"), ("q_weight", _vp),
                ("k_weight", _vp), ("positions", _vp), ("table", _vp), ("slots", _vp), ("places", _i64),
                ("cache_rows", _i64), ("tokens", _i32), ("heads", _i32), ("kv_heads", _i32), ("dim", _i32),
                ("rot", _i32), ("type", _i32), ("interleaved", _i32), ("eps", _f32)]


class CacheRef(C.Structure):
    """include/pc_hip.h CacheRef."""
    _fields_ = [("start", _vp), ("pages", _vp), ("pages_seq", _i64), ("width", _i32), ("page_rows", _i32)]


class AttentionArgs(C.Structure):
    """include/pc_hip.h AttentionArgs."""
    _fields_ = [*_ref("q"), *_ref("k"), *_ref("v"), *_ref("out"), ("lse", _vp), ("q_start", _vp), ("k_start", _vp),
                ("k_len", _vp), ("work", _vp), ("work_bytes", C.c_uint64), ("kv_rows", _i64), ("tokens", _i32),
                ("seqs", _i32), ("heads", _i32), ("kv_heads", _i32), ("dim", _i32), ("type", _i32), ("causal", _i32),
                ("max_q", _i32), ("max_k", _i32), ("scale", _f32)]


class AttentionPagedArgs(C.Structure):
    """include/pc_hip.h AttentionPagedArgs."""
    _fields_ = [("attention", AttentionArgs), ("cache", CacheRef)]


class KeyWeightsArgs(C.Structure):
    """include/pc_hip.h KeyWeightsArgs."""
    _fields_ = [*_ref("q"), *_ref("k"), *_ref("weights"), *_ref("before"), *_ref("places"), ("cache", CacheRef), ("lse", _vp),
                ("q_start", _vp), ("k_len", _vp), ("next_place", _vp), ("work", _vp), ("work_bytes", C.c_uint64), ("kv_rows", _i64),
                ("tokens", _i32), ("seqs", _i32), ("heads", _i32), ("kv_heads", _i32), ("dim", _i32), ("type", _i32),
                ("causal", _i32), ("max_q", _i32), ("max_k", _i32), ("scale", _f32), ("decay", _f32), ("pad", _i32)]


class EvictArgs(C.Structure):
    """include/pc_hip.h EvictArgs."""
    _fields_ = [*_ref("weights"), *_ref("places"), ("cache", CacheRef), ("k_len", _vp), ("next_place", _vp), ("moves", _vp),
                ("count", _vp), ("kept_len", _vp), ("work", _vp), ("work_bytes", C.c_uint64), ("rows", _i64), ("seqs", _i32), ("kv_heads", _i32), ("keep", _i32),
                ("recent", _i32), ("first", _i32), ("most", _i32), ("max_k", _i32), ("pad", _i32)]


class HeadsRef(C.Structure):
    """include/pc_hip.h HeadsRef."""
    _fields_ = [("base", _vp), ("token", _i64), ("head", _i64)]


class MoveRowsArgs(C.Structure):
    """include/pc_hip.h MoveRowsArgs."""
    _fields_ = [("t", HeadsRef * 4), ("cache", CacheRef), ("moves", _vp), ("count", _vp), ("rows", _i64), ("size", _i32 * 4),
                ("dim", _i32 * 4), ("tensors", _i32), ("seqs", _i32), ("kv_heads", _i32), ("most", _i32)]


# the same layouts for struct.pack: a call packs its arguments in about a microsecond, a ctypes Structure takes four
_ROTARY = struct.Struct("@" + "Pqq" * 2 + "PPq" + "i" * 8)
_QK_NORM_ROTARY = struct.Struct("@" + "Pqq" * 6 + "P" * 5 + "qq" + "i" * 7 + "f")
_ATTENTION = struct.Struct("@" + "Pqq" * 4 + "P" * 5 + "Qq" + "i" * 9 + "f")
_CACHE = struct.Struct("@PPqii")
_KEY_WEIGHTS = struct.Struct("@" + "Pqq" * 5 + "PPqii" + "P" * 5 + "Qq" + "i" * 9 + "ffi")
_EVICT = struct.Struct("@" + "Pqq" * 2 + "PPqii" + "P" * 6 + "Qq" + "i" * 8)
_MOVE_ROWS = struct.Struct("@" + "Pqq" * 4 + "PPqii" + "PPq" + "i" * 12)
assert (_ROTARY.size, _QK_NORM_ROTARY.size, _ATTENTION.size) == (104, 232, 192)
assert _CACHE.size == C.sizeof(CacheRef) == 32
assert _KEY_WEIGHTS.size == C.sizeof(KeyWeightsArgs) == 256
assert (_EVICT.size, C.sizeof(EvictArgs), _MOVE_ROWS.size, C.sizeof(MoveRowsArgs)) == (176, 176, 200, 200)
assert (C.sizeof(RotaryArgs), C.sizeof(QkNormRotaryArgs), C.sizeof(AttentionArgs)) == (104, 232, 192)


def _heads(x, name):
    """(address, token stride, head stride, shape, type) of a tensor [tokens][heads][dim]"""
    shape, st = x.shape, x.stride()
    if len(shape) != 3:
        raise ValueError(f"{name}: a tensor [tokens][heads][dim] is wanted, got {tuple(shape)}")
    if not x.is_cuda:
        raise ValueError(f"{name}: not on the device")
    if st[2] != 1 and shape[2] > 1:
        raise ValueError(f"{name}: its last dimension is not dense")
    return x.data_ptr(), st[0], st[1], shape, _known.get(x.dtype) or _type(x.dtype)


def _flat(x, name, dtype, count):
    """the address of a dense tensor of `count` values (None: any number) of one type"""
    if not x.is_cuda:
        raise ValueError(f"{name}: not on the device")
    if (_known.get(x.dtype) or _type(x.dtype)) != dtype:
        raise ValueError(f"{name}: {dtype} is wanted, got {x.dtype}")
    if not x.is_contiguous():
        raise ValueError(f"{name}: not dense")
    if count is not None and x.numel() != count:
        raise ValueError(f"{name}: {count} values are wanted, got {x.numel()}")
    return x.data_ptr()


def _layout(layout):
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout {layout}: half or interleaved")
    return layout == "interleaved"


def _table(table, positions, tokens):
    """(positions' address, table's address, places, rot)"""
    if table is None:
        return 0, 0, 0, 0
    if len(table.shape) != 3 or table.shape[2] != 2:
        raise ValueError("table: [places][rot / 2][2] is wanted")
    return (_flat(positions, "positions", "i32", tokens), _flat(table, "table", "f32", None), table.shape[0],
            2 * table.shape[1])


def _pages(pages, page_rows, seqs):
    """(address, distance of two sequences' tables, width) of a table of pages [seqs][width]"""
    if not pages.is_cuda:
        raise ValueError("pages: not on the device")
    if (_known.get(pages.dtype) or _type(pages.dtype)) != "i32" or len(pages.shape) != 2:
        raise ValueError("pages: a table [sequences][pages] of i32 is wanted")
    n, width = pages.shape
    step, inner = pages.stride()
    if n != seqs or width < 1 or (inner != 1 and width > 1):
        raise ValueError(f"pages: a row of pages for each of {seqs} sequences, dense, is wanted")
    if page_rows < 16 or page_rows & (page_rows - 1):
        raise ValueError(f"page_rows {page_rows}: a power of two, 16 or more")
    return pages.data_ptr(), step if n > 1 else width, width


def _cache(k_start, pages, page_rows, seqs):
    """CacheRef's fields: one run of rows for each sequence, or its pages"""
    if (k_start is None) == (pages is None) or (pages is None) != (page_rows is None):
        raise ValueError("k_start, or pages and page_rows: one of them says where the keys lie")
    if pages is None:
        return _flat(k_start, "k_start", "i64", seqs), 0, 0, 0, 0
    ptr, step, width = _pages(pages, page_rows, seqs)
    return 0, ptr, step, width, page_rows


def _per_key(x, name, dtype, shape=None):
    """(address, row stride, head stride) of a tensor [rows][kv heads] (of this shape, if given), by any strides"""
    if not x.is_cuda:
        raise ValueError(f"{name}: not on the device")
    if (_known.get(x.dtype) or _type(x.dtype)) != dtype or len(x.shape) != 2:
        raise ValueError(f"{name}: {dtype} [rows][kv heads] is wanted, got {x.dtype} {tuple(x.shape)}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name}: {tuple(shape)} is wanted, got {tuple(x.shape)}")
    return (x.data_ptr(), *x.stride())


def block_checked(heads, kv_heads, dim, capacity, dtype, table, layout, q_weight, k_weight):
    """ValueError for what a block of these sizes could not be appended to, or only with NaN in its cache."""
    if _type(dtype) not in ("bf16", "f16") or not 8 <= dim <= 256 or dim % 8:
        raise ValueError(f"{dim} dimensions of {dtype}: attention takes bf16 and f16, a multiple of 8 up to 256")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads on {kv_heads} key heads: a whole number each")
    if capacity < 1:
        raise ValueError("capacity: one token or more")
    _layout(layout)
    if table is not None:
        if len(table.shape) != 3 or table.shape[2] != 2 or 2 * table.shape[1] > dim or table.shape[0] < capacity:
            raise ValueError(f"table: [places][rot / 2][2] with {capacity} places or more and rot up to {dim} is wanted")
        _flat(table, "table", "f32", None)
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _flat(w, name, "f32", dim)


class Clear:
    """The operators on one stream, with a workspace of `workspace` bytes for attention that splits its keys. One Clear
    serves one stream at a time; its calls do not synchronise."""

    def __init__(self, stream, workspace=64 << 20):
        self.stream = stream
        self.work = DevBuf(-(-int(workspace) // 4)) if workspace else None
        if workspace:
            self.work.zero()  # the counters of split attention: zero before the first call, and left so by every call
        self._work = (self.work.ptr.value, 4 * self.work.words) if workspace else (0, 0)

    def rotary(self, x, positions, table, out, layout="half", inverse=False):
        """out = x [tokens][heads][dim] with the first rot dimensions of each head turned by table[positions[t]] (f32
        [places][rot / 2][2], rotary_table), or back where inverse; layout: pairs (i, i + rot / 2) ("half") or (2 i,
        2 i + 1) ("interleaved"). out may be x."""
        a, at, ah, shape, kind = _heads(x, "x")
        b, bt, bh, oshape, okind = _heads(out, "out")
        tokens, heads, dim = shape
        if oshape != shape or okind != kind or kind not in TYPES:
            raise ValueError("x and out: one shape and one floating type")
        pos, tab, places, rot = _table(table, positions, tokens)
        args = _ROTARY.pack(a, at, ah, b, bt, bh, pos, tab, places, tokens, heads, dim, rot, TYPES[kind], _layout(layout),
                            bool(inverse), 0)
        check(LIB.pcx_rotary(args, self.stream.h), "rotary")

    def qk_norm_rotary(self, q, k, q_weight, k_weight, positions, table, q_out, k_out, eps=1e-6, layout="half", v=None,
                       v_out=None, slots=None):
        """q_out and k_out = the heads of q and k [tokens][heads][dim], each x w / sqrt(mean(x^2) + eps) (weights f32 [dim]
        or None for ones), then turned as by rotary (table None: not turned). slots (i64 [tokens]): row t of k goes to
        row slots[t] of k_out, a cache, and v's row (if given) to that of v_out; slots outside it are not written."""
        a, at, ah, qs, kind = _heads(q, "q")
        b, bt, bh, ks, kkind = _heads(k, "k")
        c, ct, ch, qos, qok = _heads(q_out, "q_out")
        d, dt, dh, kos, kok = _heads(k_out, "k_out")
        tokens, heads, dim = qs
        kv = ks[1]
        if ks[0] != tokens or ks[2] != dim or qos != qs or kos[1:] != ks[1:]:
            raise ValueError("q and k: the same tokens and dim, the outputs' shapes as theirs")
        if not kind == kkind == qok == kok or kind not in TYPES:
            raise ValueError("q, k and the outputs: one floating type")
        if slots is None and kos[0] != tokens:
            raise ValueError("k_out: one row for each token where there are no slots")
        e, et, eh, f, ft, fh = 0, 0, 0, 0, 0, 0
        if (v is None) != (v_out is None):
            raise ValueError("v and v_out go together")
        if v is not None:
            e, et, eh, vs, vk = _heads(v, "v")
            f, ft, fh, vos, vok = _heads(v_out, "v_out")
            if vs != ks or vos != kos or not vk == vok == kind:
                raise ValueError("v and v_out: the shapes and type of k and k_out")
        pos, tab, places, rot = _table(table, positions, tokens)
        args = _QK_NORM_ROTARY.pack(
            a, at, ah, b, bt, bh, e, et, eh, c, ct, ch, d, dt, dh, f, ft, fh,
            0 if q_weight is None else _flat(q_weight, "q_weight", "f32", dim),
            0 if k_weight is None else _flat(k_weight, "k_weight", "f32", dim), pos, tab,
            0 if slots is None else _flat(slots, "slots", "i64", tokens), places, kos[0], tokens, heads, kv, dim, rot,
            TYPES[kind], _layout(layout), eps)
        check(LIB.pcx_qk_norm_rotary(args, self.stream.h), "qk_norm_rotary")

    def attention(self, q, k, v, q_start, k_start, k_len, out, lse=None, scale=None, causal=True, max_q=None, max_k=None):
        """out [tokens][heads][dim] and lse (f32 [tokens][heads], or None) of the packed queries q over k and v [rows][kv
        heads][dim]: sequence b has q's rows q_start[b] .. q_start[b + 1] - 1 (i32) and k's k_start[b] .. + k_len[b] - 1
        (i64, i32; device arrays). causal: the last query sees the last key, each earlier one a key less. scale: 1 /
        sqrt(dim) unless given. max_q, max_k: the longest runs expected (the buffers' rows unless given); they only
        choose kernels, which differ in the order of their sums and in whether what the weights' rounding to the type leaves
        is added (it is for tokens)."""
        args = self._attention(q, k, v, q_start, k_start, k_len, out, lse, scale, causal, max_q, max_k)
        check(LIB.pcx_attention(args, self.stream.h), "attention")

    def attention_args(self, *args, **kw):
        """attention's checked arguments as the struct that pcx_attention and pcx_attention_workspace take."""
        return AttentionArgs.from_buffer_copy(self._attention(*args, **kw))

    def attention_paged(self, q, k, v, q_start, pages, page_rows, k_len, out, lse=None, scale=None, causal=True, max_q=None,
                        max_k=None):
        """attention over keys and values in pages: k and v [rows][kv heads][dim] are pools of rows / page_rows pages (page_rows:
        a power of two, 16 or more), sequence b has the first k_len[b] keys of the pages pages[b] (i32 [sequences][width], any
        order, shared or not): key j in row pages[b][j / page_rows] page_rows + j % page_rows, the slot that qk_norm_rotary
        writes it to."""
        args = self._attention_paged(q, k, v, q_start, pages, page_rows, k_len, out, lse, scale, causal, max_q, max_k)
        check(LIB.pcx_attention_paged(args, self.stream.h), "attention_paged")

    def attention_paged_args(self, *args, **kw):
        """attention_paged's checked arguments as the struct that pcx_attention_paged and its workspace query take."""
        return AttentionPagedArgs.from_buffer_copy(self._attention_paged(*args, **kw))

    def _attention_paged(self, q, k, v, q_start, pages, page_rows, k_len, out, lse=None, scale=None, causal=True, max_q=None,
                         max_k=None):
        ptr, step, width = _pages(pages, page_rows, k_len.shape[0])
        room = min(width * page_rows, 0x7FFFFFFF)
        max_k = room if max_k is None else min(max_k, room)
        return self._attention(q, k, v, q_start, None, k_len, out, lse, scale, causal, max_q, max_k) + _CACHE.pack(
            0, ptr, step, width, page_rows)

    def key_weights(self, q, k, lse, q_start, k_len, weights, k_start=None, pages=None, page_rows=None, before=None, decay=1.0,
                    places=None, next_place=None, scale=None, causal=True, max_q=None, max_k=None):
        """The weight that keys gather: weights (f32 [rows][kv heads], by any strides) = decay x before (the same shape, or None
        for zeros; weights itself where they gather) + the sum of exp(scale q . k - lse) over the queries that see a key and the
        heads of its group; q, k, lse and the runs as attention took and gave them, the keys' rows from k_start on or in pages.
        next_place (i32 [sequences], the place after each sequence's last token): the last keys are the queries' own and new,
        they begin at 0, and get their places (i32 [rows][kv heads], if given). Sequences may not share rows. max_q, max_k: the
        longest runs expected; they only choose how rows are split."""
        args = self._key_weights(q, k, lse, q_start, k_len, weights, k_start, pages, page_rows, before, decay, places, next_place,
                                 scale, causal, max_q, max_k)
        check(LIB.pcx_key_weights(args, self.stream.h), "key_weights")

    def key_weights_args(self, *args, **kw):
        """key_weights' checked arguments as the struct that pcx_key_weights and its workspace query take."""
        return KeyWeightsArgs.from_buffer_copy(self._key_weights(*args, **kw))

    def _key_weights(self, q, k, lse, q_start, k_len, weights, k_start=None, pages=None, page_rows=None, before=None, decay=1.0,
                     places=None, next_place=None, scale=None, causal=True, max_q=None, max_k=None):
        a, at, ah, qs, kind = _heads(q, "q")
        b, bt, bh, ks, kkind = _heads(k, "k")
        tokens, heads, dim = qs
        rows, kv, kdim = ks
        if kdim != dim or kind != kkind or kind not in TYPES:
            raise ValueError("q and k: one dim, one floating type")
        if places is not None and next_place is None:
            raise ValueError("places: next_place says where they go on")
        seqs = k_len.shape[0]
        cache = _cache(k_start, pages, page_rows, seqs)
        room = rows if pages is None else min(rows, cache[3] * page_rows)
        none = (0, 0, 0)
        return _KEY_WEIGHTS.pack(
            a, at, ah, b, bt, bh, *_per_key(weights, "weights", "f32", (rows, kv)),
            *(none if before is None else _per_key(before, "before", "f32", (rows, kv))),
            *(none if places is None else _per_key(places, "places", "i32", (rows, kv))), *cache,
            _flat(lse, "lse", "f32", tokens * heads), _flat(q_start, "q_start", "i32", seqs + 1), _flat(k_len, "k_len", "i32", seqs),
            0 if next_place is None else _flat(next_place, "next_place", "i32", seqs), *self._work, rows, tokens, seqs, heads, kv, dim,
            TYPES[kind], bool(causal), tokens if max_q is None else max_q, min(room if max_k is None else max_k, 0x7FFFFFFF),
            dim ** -0.5 if scale is None else scale, decay, 0)

    def evict(self, weights, k_len, keep, moves, count, k_start=None, pages=None, page_rows=None, places=None, next_place=None,
              recent=0, first=0, kept_len=None, max_k=None):
        """Which keys leave: each key head of a sequence keeps the `keep` of its k_len[b] keys with the largest weights (f32
        [rows][kv heads], by any strides), the lower key of two alike; before all others those whose place (i32, as the weights;
        None: the key's number) is below `first` or at least next_place[b] (i32; None: the length) - recent, `keep` of them at
        most. moves (i32 [sequences][kv heads][most][2]) and count (i32 [sequences][kv heads]) get the rows that move_rows moves,
        kept keys from behind `keep` to the gaps before it; kept_len (i32, or None) the lengths after that. Moves past `most` are
        not written (there are never more than keep, or than the longest run less keep). max_k: the longest run expected; it only
        chooses a kernel."""
        seqs = k_len.shape[0]
        rows, kv = weights.shape if len(weights.shape) == 2 else (0, 0)
        shape = moves.shape
        if len(shape) != 4 or shape[0] != seqs or shape[1] != kv or shape[3] != 2:
            raise ValueError(f"moves: [{seqs}][{kv}][most][2] is wanted, got {tuple(shape)}")
        if min(keep, recent, first) < 0 or first + recent > keep:
            raise ValueError(f"keep {keep}, recent {recent}, first {first}: none negative, no more protected than kept")
        w = _per_key(weights, "weights", "f32")
        p = (0, 0, 0) if places is None else _per_key(places, "places", "i32", (rows, kv))
        cache = _cache(k_start, pages, page_rows, seqs)
        room = rows if pages is None else cache[3] * page_rows
        args = _EVICT.pack(
            *w, *p, *cache, _flat(k_len, "k_len", "i32", seqs),
            0 if next_place is None else _flat(next_place, "next_place", "i32", seqs),
            _flat(moves, "moves", "i32", None), _flat(count, "count", "i32", seqs * kv),
            0 if kept_len is None else _flat(kept_len, "kept_len", "i32", seqs), *self._work, rows, seqs, kv, keep, recent, first, shape[2],
            min(room if max_k is None else max_k, 0x7FFFFFFF), 0)
        check(LIB.pcx_evict(args, self.stream.h), "evict")

    def move_rows(self, moves, count, tensors, k_start=None, pages=None, page_rows=None):
        """The moves that evict chose, in up to four tensors [rows][kv heads][dim] or [rows][kv heads] of any types at once, by any
        strides of rows and heads: keys, values, their weights and places. Rows move in place, all moves at once; sequences may
        not share rows."""
        shape = moves.shape
        if len(shape) != 4 or shape[3] != 2 or not 1 <= len(tensors) <= 4:
            raise ValueError("moves [sequences][kv heads][most][2], and one to four tensors")
        seqs, kv, most, _ = shape
        refs, sizes, dims, rows = [], [], [], None
        for x in tensors:
            kind = _known.get(x.dtype) or _type(x.dtype)
            if len(x.shape) == 2:
                refs += _per_key(x, "tensors", kind)
                (r, heads), dim = x.shape, 1
            else:
                at, row, head, (r, heads, dim), _ = _heads(x, "tensors")
                refs += at, row, head
            if heads != kv or rows not in (None, r):
                raise ValueError(f"tensors: the same rows and {kv} key heads each")
            rows = r
            dims.append(dim)
            sizes.append(SIZES[kind])
        n = 4 - len(tensors)
        args = _MOVE_ROWS.pack(*refs, *[0] * 3 * n, *_cache(k_start, pages, page_rows, seqs), _flat(moves, "moves", "i32", None),
                               _flat(count, "count", "i32", seqs * kv), rows, *sizes, *[0] * n, *dims, *[0] * n, len(tensors), seqs, kv,
                               most)
        check(LIB.pcx_move_rows(args, self.stream.h), "move_rows")

    def _attention(self, q, k, v, q_start, k_start, k_len, out, lse=None, scale=None, causal=True, max_q=None, max_k=None):
        a, at, ah, qs, kind = _heads(q, "q")
        b, bt, bh, ks, kkind = _heads(k, "k")
        c, ct, ch, vs, vkind = _heads(v, "v")
        d, dt, dh, os, okind = _heads(out, "out")
        tokens, heads, dim = qs
        rows, kv, kdim = ks
        if kdim != dim or vs != ks or os != qs:
            raise ValueError("k and v alike, out as q, one dim")
        if not kind == kkind == vkind == okind or kind not in TYPES:
            raise ValueError("q, k, v and out: one floating type")
        seqs = k_len.shape[0]
        return _ATTENTION.pack(
            a, at, ah, b, bt, bh, c, ct, ch, d, dt, dh, 0 if lse is None else _flat(lse, "lse", "f32", tokens * heads),
            _flat(q_start, "q_start", "i32", seqs + 1), 0 if k_start is None else _flat(k_start, "k_start", "i64", seqs),
            _flat(k_len, "k_len", "i32", seqs), *self._work, rows, tokens, seqs, heads, kv, dim, TYPES[kind],
            bool(causal), tokens if max_q is None else max_q, min(rows, 0x7FFFFFFF) if max_k is None else max_k,
            dim ** -0.5 if scale is None else scale)
