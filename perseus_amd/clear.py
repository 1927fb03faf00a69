"""The clear side of an encrypted transformer block, on the device: rotary positions, the norms of queries and keys with
the rotation in the same pass, and attention over packed prompts, chunks and single tokens.

The encrypted scoring (perseus_amd.attention) multiplies plaintext queries into an encrypted cache of keys. `Clear` makes
those queries and keys from projected rows, and the attention in the clear that the decrypted scores are held against: its
log-sum-exp turns a score into a probability, exp(score - lse). The kernels are csrc/rotary.hip and csrc/attend.hip behind
pcx_rotary, pcx_qk_norm_rotary and pcx_attention (include/pc_hip.h), which a C caller uses directly.

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


class AttentionArgs(C.Structure):
    """include/pc_hip.h AttentionArgs."""
    _fields_ = [*_ref("q"), *_ref("k"), *_ref("v"), *_ref("out"), ("lse", _vp), ("q_start", _vp), ("k_start", _vp),
                ("k_len", _vp), ("work", _vp), ("work_bytes", C.c_uint64), ("kv_rows", _i64), ("tokens", _i32),
                ("seqs", _i32), ("heads", _i32), ("kv_heads", _i32), ("dim", _i32), ("type", _i32), ("causal", _i32),
                ("max_q", _i32), ("max_k", _i32), ("scale", _f32)]


# the same layouts for struct.pack: a call packs its arguments in about a microsecond, a ctypes Structure takes four
_ROTARY = struct.Struct("@" + "Pqq" * 2 + "PPq" + "i" * 8)
_QK_NORM_ROTARY = struct.Struct("@" + "Pqq" * 6 + "P" * 5 + "qq" + "i" * 7 + "f")
_ATTENTION = struct.Struct("@" + "Pqq" * 4 + "P" * 5 + "Qq" + "i" * 9 + "f")
assert (_ROTARY.size, _QK_NORM_ROTARY.size, _ATTENTION.size) == (104, 232, 192)
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
            _flat(q_start, "q_start", "i32", seqs + 1), _flat(k_start, "k_start", "i64", seqs),
            _flat(k_len, "k_len", "i32", seqs), *self._work, rows, tokens, seqs, heads, kv, dim, TYPES[kind],
            bool(causal), tokens if max_q is None else max_q, min(rows, 0x7FFFFFFF) if max_k is None else max_k,
            dim ** -0.5 if scale is None else scale)
