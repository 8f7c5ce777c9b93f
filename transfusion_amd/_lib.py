"""ctypes binding of libtfusion_hip.so.

The ctypes ``Structure`` classes are generated by parsing ``include/tfusion.h`` at import time, so
the Python view of the C ABI cannot drift from the header.  There is NO fallback: if the shared
library is missing or a symbol is absent, importing the product path raises.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(os.path.dirname(HERE), "include", "tfusion.h")
LIB_PATH = os.environ.get("TFUSION_LIB") or os.path.join(HERE, "lib", "libtfusion_hip.so")   # override: same-box A/B of two builds

_SCALARS = {
    "int": C.c_int, "unsigned": C.c_uint, "float": C.c_float, "uint64_t": C.c_uint64, "uint32_t": C.c_uint32,
    "size_t": C.c_size_t, "long long": C.c_longlong, "uint8_t": C.c_uint8, "char": C.c_char, "double": C.c_double,
}


class TfError(RuntimeError):
    pass


def _strip_comments(text: str) -> str:
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def _parse_header(path: str):
    text = _strip_comments(open(path).read())
    consts = {m.group(1): int(m.group(2)) for m in re.finditer(r"#define\s+(TF_\w+)\s+\(?(-?\d+)\)?", text)}
    enums = {}
    for m in re.finditer(r"enum\s+\w+\s*\{(.*?)\}", text, flags=re.S):
        for item in m.group(1).split(","):
            item = item.strip()
            if item:
                k, v = item.split("=")
                enums[k.strip()] = int(v)
    structs = {}
    for m in re.finditer(r"typedef\s+struct\s+(\w+)\s*\{(.*?)\}\s*\1\s*;", text, flags=re.S):
        name, body = m.group(1), m.group(2)
        fields = []
        for stmt in body.split(";"):
            stmt = " ".join(stmt.split())
            if not stmt:
                continue
            stmt = stmt.replace("const ", "")
            # base type = longest known prefix
            base = None
            for cand in sorted(list(_SCALARS) + list(structs) + ["void"], key=len, reverse=True):
                if stmt.startswith(cand + " ") or stmt.startswith(cand + "*"):
                    base = cand
                    break
            if base is None:
                raise TfError(f"cannot parse field '{stmt}' of {name}")
            rest = stmt[len(base):]
            for decl in rest.split(","):
                decl = decl.strip()
                ptr = decl.count("*")
                decl = decl.replace("*", "").strip()
                arr = re.match(r"(\w+)\[(\w+)\]", decl)
                if base == "void" or ptr:
                    ctype = C.c_void_p
                elif base in _SCALARS:
                    ctype = _SCALARS[base]
                else:
                    ctype = structs[base]
                if arr:
                    n = arr.group(2)
                    n = consts[n] if n in consts else int(n)
                    fields.append((arr.group(1), ctype * n))
                else:
                    fields.append((decl, ctype))
        structs[name] = type(name, (C.Structure,), {"_fields_": fields})
    funcs = re.findall(r"^\s*(?:int|long long|uint32_t|float|size_t|void|const char\*|const uint32_t\*)\s+(tf_\w+)\s*\(", text, flags=re.M)
    return consts, enums, structs, sorted(set(funcs))


CONSTS, ENUMS, STRUCTS, FUNCTIONS = _parse_header(HEADER)

_CODES = {C.c_void_p: "P", C.c_int: "i", C.c_uint: "I", C.c_float: "f", C.c_double: "d", C.c_longlong: "q", C.c_size_t: "N", C.c_uint64: "Q",
          C.c_uint32: "I"}


def packer(name: str):
    """The ``pack`` of a flat argument struct: all its fields in the header's order -> the bytes the library reads (native alignment).
    Filling a ctypes structure of fifty fields by keyword costs 5 us a call, this 1 us -- it matters where the call is a single token."""
    fields = STRUCTS[name]._fields_
    st = struct.Struct("@" + "".join(_CODES[t] for _, t in fields) + "0P")
    if st.size != C.sizeof(STRUCTS[name]):
        raise TfError(f"{name} does not pack to the size of its C layout")
    return st.pack
globals().update(STRUCTS)
globals().update(ENUMS)
TF_MAX_LAYERS = CONSTS["TF_MAX_LAYERS"]

_lib = None


def load():
    """Load the shared library (once).  Raises TfError when it is missing: there is no CPU path."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise TfError(f"{LIB_PATH} not built: run `python -m transfusion_amd.build` (hipcc, gfx950). "
                      "transfusion_amd has no CPU fallback.")
    # torch ships its own libamdhip64/HSA runtime: it must be resident BEFORE our library is mapped, so that our
    # DT_NEEDED libamdhip64.so resolves to the runtime torch's streams and allocations live in (two HIP runtimes in
    # one process do not see each other's devices).
    import torch  # noqa: F401
    lib = C.CDLL(LIB_PATH)
    missing = [f for f in FUNCTIONS if not hasattr(lib, f)]
    if missing:
        raise TfError(f"libtfusion_hip.so lacks symbols declared in tfusion.h: {missing}")
    lib.tf_last_error.restype = C.c_char_p
    lib.tf_drop_key.restype = C.c_uint32
    lib.tf_drop_key.argtypes = [C.c_uint64, C.c_uint32]
    lib.tf_drop_threshold.restype = C.c_uint32
    lib.tf_drop_threshold.argtypes = [C.c_float]
    lib.tf_drop_scale.restype = C.c_float
    lib.tf_drop_scale.argtypes = [C.c_float]
    lib.tf_attn_dropmask_bytes.restype = C.c_size_t
    lib.tf_attn_dropmask_bytes.argtypes = [C.c_int] * 3
    lib.tf_clock_ptr.restype = C.c_void_p
    lib.tf_clock_ptr.argtypes = []
    lib.tf_clock_advance.argtypes = [C.c_uint32, C.c_void_p]
    lib.tf_clock_set.argtypes = [C.c_uint32, C.c_void_p]
    lib.tf_set_gemm_concurrency.restype = None
    lib.tf_set_gemm_concurrency.argtypes = [C.c_int]
    lib.tf_attn_ds_bytes.restype = C.c_size_t
    lib.tf_attn_ds_bytes.argtypes = [C.c_int] * 3
    lib.tf_attn_dropmask.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_uint32, C.c_uint32, C.c_void_p]
    lib.tf_attn_dropmask_rows.argtypes = [C.c_void_p, C.c_longlong, C.c_int, C.c_uint32, C.c_uint32, C.c_void_p]
    lib.tf_encoder_peek.restype = C.c_longlong
    lib.tf_encoder_peek.argtypes = [C.c_void_p, C.c_char_p, C.c_void_p, C.c_longlong, C.c_void_p]
    lib.tf_encoder_plan.argtypes = [C.c_int] * 7 + [C.c_void_p]
    lib.tf_encoder_plan_ex.argtypes = [C.c_void_p, C.c_void_p]
    lib.tf_softplus_col.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
    lib.tf_quant_rows_fp8.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_void_p]
    lib.tf_attn_block_skip.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
    lib.tf_debug_spin.argtypes = [C.c_int, C.c_void_p]
    lib.tf_trace_stop.restype = C.c_longlong
    lib.tf_trace_stop.argtypes = [C.c_void_p, C.c_longlong]
    for f in ("tf_sumsq", "tf_sumsq_set"):
        getattr(lib, f).argtypes = [C.c_void_p, C.c_longlong, C.c_void_p, C.c_void_p]
    lib.tf_score_attn_work.restype = C.c_size_t
    lib.tf_score_attn_work.argtypes = [C.c_int] * 7
    lib.tf_score_attn_bwd_work.restype = C.c_size_t
    lib.tf_score_attn_bwd_work.argtypes = [C.c_int] * 8
    lib.tf_grad_clip_parts.restype = C.c_longlong
    lib.tf_grad_clip_parts.argtypes = [C.c_void_p, C.c_int]
    lib.tf_dropout_mask.argtypes = [C.c_void_p, C.c_longlong, C.c_uint32, C.c_uint32, C.c_void_p]
    lib.tf_dropout_apply.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_uint32, C.c_uint32, C.c_float, C.c_void_p]
    lib.tf_cast_f32_bf16.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]
    lib.tf_cast_bf16_f32.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]
    if lib.tf_version() != CONSTS["TF_ABI_VERSION"]:
        raise TfError("ABI version mismatch between tfusion.h and libtfusion_hip.so")
    _lib = lib
    return lib


def check(rc: int, what: str = ""):
    if rc != 0:
        msg = load().tf_last_error().decode()
        raise TfError(f"{what or 'tfusion call'} failed (rc={rc}): {msg}")


def call(fn_name: str, args_struct, stream: int, *extra):
    """Invoke an ``int fn(const Struct*, [extra ints...], tf_stream_t)`` entry."""
    lib = load()
    fn = getattr(lib, fn_name)
    args = [C.byref(args_struct)] + [C.c_int(x) for x in extra] + [C.c_void_p(stream)]
    check(fn(*args), fn_name)


def call_packed(fn_name: str, packed: bytes, stream: int):
    """``call`` of an entry whose argument struct was formed by ``packer``."""
    rc = getattr(_lib or load(), fn_name)(packed, C.c_void_p(stream))
    if rc:
        check(rc, fn_name)


def ptr(t) -> int:
    """Device pointer of a torch tensor (0 for None)."""
    return 0 if t is None else t.data_ptr()


def current_stream() -> int:
    from transfusion_amd import ops          # (the fast raw-handle lookup lives there)
    return ops._stream()
