"""ctypes binding of libdig_hip.so (the C-ABI boundary declared in include/dig_hip.h).

The argument structs are generated from the header text itself, so the Python mirror cannot drift from
the C declarations.  There is NO fallback: if the library is missing or a call fails, this raises.
"""
import ctypes
import os
import re
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(os.path.dirname(_HERE), "include", "dig_hip.h")
LIB_PATH = os.environ.get("DIG_HIP_LIB", os.path.join(_HERE, "csrc", "libdig_hip.so"))  # override only for A/B kernel experiments

DIG_BF16, DIG_F32 = 0, 1

_SCALARS = {"int": ctypes.c_int, "float": ctypes.c_float, "long long": ctypes.c_longlong}


def _parse_header(text):
    """-> (structs {name: [(field, ctype)]}, functions [name])"""
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    structs = {}
    for body, name in re.findall(r"typedef\s+struct\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
        fields = []
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            if "*" in decl:  # pointer field(s): "const void* a" (one per declaration in this header)
                fname = decl.rsplit("*", 1)[1].strip()
                fields.append((fname, ctypes.c_void_p))
                continue
            for base in ("long long", "int", "float"):
                if decl.startswith(base + " "):
                    for item in decl[len(base):].split(","):
                        item = item.strip()
                        m = re.match(r"(\w+)\[(\d+)\]$", item)
                        if m:
                            fields.append((m.group(1), _SCALARS[base] * int(m.group(2))))
                        else:
                            fields.append((item, _SCALARS[base]))
                    break
            else:
                raise RuntimeError(f"dig_hip.h: cannot parse field declaration {decl!r}")
        structs[name] = fields
    funcs = re.findall(r"^\s*(?:int|const char\*)\s+(dig_\w+)\s*\(", text, flags=re.M)
    return structs, funcs


with open(HEADER) as _f:
    _STRUCT_FIELDS, FUNCTIONS = _parse_header(_f.read())

STRUCTS = {}
for _name, _fields in _STRUCT_FIELDS.items():
    STRUCTS[_name] = type(_name, (ctypes.Structure,), {"_fields_": _fields})

_lib = None


def lib():
    """Load the shared library (once).  Raises if it has not been built - never falls back."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} not found: build it with `make -C dig_amd/csrc` (or __graft_entry__.build()). "
                "dig_amd has no CPU fallback.")
        L = ctypes.CDLL(LIB_PATH)
        for fn in FUNCTIONS:
            f = getattr(L, fn)  # AttributeError if a declared symbol is not exported
            f.restype = ctypes.c_char_p if fn == "dig_last_error" else ctypes.c_int
        _lib = L
    return _lib


def _ptr(x):
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()  # torch.Tensor


_SNAME = {"gemm_nt": "dig_gemm_args", "qsample_stem": "dig_stem_args", "bilinear_ac_concat": "dig_bilinear_ac_args",
          "nchw_f32_to_nhwc": "dig_layout_args", "nhwc_to_nchw_f32": "dig_layout_args"}
_FMT = {ctypes.c_void_p: "P", ctypes.c_int: "i", ctypes.c_float: "f", ctypes.c_longlong: "q"}


class _Entry:
    """dig_<fn> and how its argument block is packed: one struct.pack of all fields in order (the per-launch host cost is what bounds
    small batches: setting the fields of a ctypes structure one by one took longer than the rest of a call)."""

    __slots__ = ("slot", "blank", "pack", "func", "name", "sname")

    def __init__(self, fn):
        S = STRUCTS[_SNAME.get(fn, f"dig_{fn}_args")]
        self.name, self.sname, self.slot, self.blank, fmt = fn, S.__name__, {}, [], ""
        for name, t in S._fields_:
            n = getattr(t, "_length_", 0)
            self.slot[name] = (len(self.blank), n, t is ctypes.c_void_p)
            self.blank += [0] * (n or 1)
            fmt += _FMT[t._type_] * n if n else _FMT[t]
        packer = struct.Struct(fmt + "0q")  # native alignment, as the C compiler lays the fields out
        if packer.size != ctypes.sizeof(S):
            raise RuntimeError(f"{self.sname}: packed size {packer.size} but the C layout has {ctypes.sizeof(S)}")
        self.pack = packer.pack
        self.func = lib()["dig_" + fn]  # a function object of its own: the block goes over as bytes
        self.func.argtypes, self.func.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int

    def refuse(self, err):
        """what struct.pack raised for a value that its field does not take, as the error of a call"""
        if "required argument" in str(err):  # of another type than the field's
            return TypeError(f"dig_{self.name}: a field of {self.sname} was given a value of the wrong type ({err})")
        return ValueError(f"dig_{self.name}: a size or pitch is larger than the kernels take ({err})")


_ENTRIES = {}


TRACE = None  # bench.py's per-launch HIP-event hook: callable(fn, kw, phase) with phase 0 before / 1 after the launch


def call(fn, stream=None, **kw):
    """Call `int dig_<fn>(const dig_<fn>_args*, void* stream)` with keyword fields; tensors become pointers.
    The launch goes to the device the tensor arguments live on (they must all share one HIP device; CPU tensors and
    mixed devices raise before anything is launched), on that device's current torch stream unless `stream` is given.
    Raises RuntimeError on a non-zero return."""
    import torch

    e = _ENTRIES.get(fn)
    if e is None:
        e = _ENTRIES[fn] = _Entry(fn)
    dev = None
    vals = e.blank[:]
    slot = e.slot
    for k, v in kw.items():
        at = slot.get(k)
        if at is None:
            raise TypeError(f"{e.sname} has no field {k!r}")
        i, n, pointer = at
        if isinstance(v, torch.Tensor):
            if not v.is_cuda:
                raise RuntimeError(f"dig_{fn}: argument {k!r} is a {v.device} tensor; the kernels take HIP-device pointers only "
                                   "(no CPU fallback) - move the module and its inputs to the device first")
            d = v.device
            if dev is None:
                dev = d
            elif d != dev:
                raise RuntimeError(f"dig_{fn}: argument {k!r} lives on {d} but another argument on {dev}")
            if not pointer:
                raise TypeError(f"dig_{fn}: {k!r} is a number, not a tensor")
            vals[i] = v.data_ptr()
        elif n:
            v = tuple(v)
            if len(v) > n:
                raise IndexError(f"dig_{fn}: {k!r} holds {n} values, got {len(v)}")
            vals[i:i + len(v)] = v
        elif v is not None:
            vals[i] = v
        elif not pointer:
            raise TypeError(f"dig_{fn}: {k!r} is a number, not None")
    try:
        block = e.pack(*vals)
    except struct.error as err:
        raise e.refuse(err) from None
    tr = TRACE
    if tr is not None:
        tr(fn, kw, 0)
    cur = torch.cuda.current_device()
    if dev is None or dev.index in (None, cur):
        rc = e.func(block, torch._C._cuda_getCurrentRawStream(cur) if stream is None else stream)
    else:  # tensors on a device that is not current: the launchers key their per-device state on hipGetDevice()
        with torch.cuda.device(dev):
            rc = e.func(block, torch._C._cuda_getCurrentRawStream(dev.index) if stream is None else stream)
    if rc != 0:
        raise RuntimeError(f"dig_{fn} failed ({rc}): {lib().dig_last_error().decode()}")
    if tr is not None:
        tr(fn, kw, 1)


def launch(fn, dev, *vals):
    """Launch dig_<fn> with its argument block's values in field order (pointers as integers, 0 = NULL), for wrappers that have checked their
    tensors already: they live on HIP device number `dev`.  The stream is that device's current one."""
    import torch

    e = _ENTRIES.get(fn)
    if e is None:
        e = _ENTRIES[fn] = _Entry(fn)
    try:
        block = e.pack(*vals)
    except struct.error as err:
        raise e.refuse(err) from None
    tr = TRACE
    if tr is not None:
        kw = dict(zip(e.slot, vals))
        tr(fn, kw, 0)
    if dev == torch._C._cuda_getDevice():
        rc = e.func(block, torch._C._cuda_getCurrentRawStream(dev))
    else:  # the launchers key their per-device state on hipGetDevice()
        with torch.cuda.device(dev):
            rc = e.func(block, torch._C._cuda_getCurrentRawStream(dev))
    if rc != 0:
        raise RuntimeError(f"dig_{fn} failed ({rc}): {lib().dig_last_error().decode()}")
    if tr is not None:
        tr(fn, kw, 1)


def dtype_code(torch_dtype):
    import torch

    if torch_dtype == torch.bfloat16:
        return DIG_BF16
    if torch_dtype == torch.float32:
        return DIG_F32
    raise ValueError(f"unsupported dtype {torch_dtype}; the HIP path stores activations as bfloat16 or float32")


def _tver(t):
    """Version counter of a tensor, 0 for an inference tensor: tensors created under torch.inference_mode() (the reference
    decorates sample_from_t / ddim_sample_from_t with it, ddp.py:770,827) track no version and raise on `_version`; they
    cannot be written in place outside inference mode either, so a constant is a sound stand-in for the cache key."""
    return 0 if t.is_inference() else t._version


def _pver(params):
    """Sum of the parameters' version counters (the re-pack key); inference tensors count 0, see _tver."""
    return sum(_tver(q) for q in params)
