#!/usr/bin/env python3
"""Generates src/backend/cuda/ffi.rs — the `extern "C"` block of the Rust binding — from include/sage_cuda.h, so
that the two cannot drift apart: every function the header declares becomes one Rust declaration with the same
name, argument order and widths.  `python bindings/rust/gen_ffi.py` rewrites the file; `--check` only compares
(tests/test_rust_binding.py runs that)."""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "sage_cuda.h")
OUT = os.path.join(HERE, "src", "backend", "cuda", "ffi.rs")

SCALARS = {"sage_status": "i32", "int32_t": "i32", "int64_t": "i64", "uint64_t": "u64", "uint32_t": "u32", "uint8_t": "u8",
           "size_t": "usize", "float": "f32", "double": "f64", "char": "c_char", "void": "c_void"}
OPAQUE = ["sage_ctx", "sage_buf", "sage_module"]
STRUCTS = ["sage_tensor", "sage_ctx_opts", "sage_mem_stats_t", "sage_arg", "sage_window", "sage_adamw_tensor", "sage_adamw_opts"]

PRELUDE = '''// GENERATED by bindings/rust/gen_ffi.py from include/sage_cuda.h — do not edit by hand.
//
// The raw C ABI of libsagecuda.so.  Safe wrappers live in backend/cuda/mod.rs.
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_void};

#[repr(C)] pub struct sage_ctx { _p: [u8; 0] }
#[repr(C)] pub struct sage_buf { _p: [u8; 0] }
#[repr(C)] pub struct sage_module { _p: [u8; 0] }

pub const SAGE_MAX_DIMS: usize = 8;
pub const SAGE_OK: i32 = 0;
pub const SAGE_ERR_INVALID: i32 = 1;
pub const SAGE_ERR_OOM: i32 = 2;
pub const SAGE_ERR_DEVICE: i32 = 3;
pub const SAGE_ERR_COMPILE: i32 = 4;
pub const SAGE_ERR_NO_DEVICE: i32 = 5;
pub const SAGE_ERR_TIMEOUT: i32 = 6;
pub const SAGE_ERR_UNSUPPORTED: i32 = 7;
pub const SAGE_F32: i32 = 0;
pub const SAGE_I32: i32 = 1;
pub const SAGE_U32: i32 = 2;
// storage types of the language-model operators alone
pub const SAGE_F16: i32 = 3;
pub const SAGE_BF16: i32 = 4;
pub const SAGE_I8: i32 = 5;
pub const SAGE_U8: i32 = 6;

/// Tensor = buffer + Shape{extents, strides, offset} in elements (src/tensor.rs:106-110, src/shape.rs:37-43).
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_tensor {
    pub buf: *mut sage_buf, pub dtype: i32, pub ndim: i32,
    pub extents: [i64; SAGE_MAX_DIMS], pub strides: [i64; SAGE_MAX_DIMS], pub offset: i64,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_ctx_opts {
    pub mem_capacity_bytes: u64, pub use_cache: i32, pub ref_compat: i32, pub pattern_fusion: i32, pub gemm_backend: i32,
}
#[repr(C)] #[derive(Clone, Copy, Default)]
pub struct sage_mem_stats_t { pub capacity: u64, pub mem_total: u64, pub mem_used: u64, pub mem_peak: u64, pub num_device_allocs: u64 }
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_arg { pub kind: i32, pub buf: *mut sage_buf, pub i: i64, pub f: f32, pub bytes: *const c_void, pub nbytes: usize }
/// Every pair is ordered [w, h] like SizedExtent<2> (src/ops/conv.rs:83).
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_window { pub ker: [i32; 2], pub stride: [i32; 2], pub pad: [i32; 2], pub dil: [i32; 2] }
/// One tensor of an AdamW step; absent operands have a null `buf`.
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_adamw_tensor {
    pub param: sage_tensor, pub grad: sage_tensor, pub m: sage_tensor, pub v: sage_tensor, pub m_scale: sage_tensor, pub v_scale: sage_tensor, pub copy: sage_tensor,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct sage_adamw_opts { pub lr: f64, pub beta1: f64, pub beta2: f64, pub eps: f64, pub weight_decay: f64, pub grad_scale: f64, pub step: i64 }

#[link(name = "sagecuda")]
extern "C" {
'''


def rust_type(ctype, array):
    t = ctype.strip()
    const = t.startswith("const ")
    t = t[6:].strip() if const else t
    stars = t.count("*")
    base = t.replace("*", "").replace("const", "").strip()
    r = SCALARS.get(base, base)
    if base not in SCALARS and base not in OPAQUE and base not in STRUCTS:
        raise SystemExit("gen_ffi: unknown C type %r" % ctype)
    if array:  # `T name[n]` decays to a pointer
        stars += 1
    if stars == 0:
        return r
    # `const T *` -> *const T; `T *const *` and `T **` -> pointer to mutable pointer
    out = r
    for level in range(stars):
        out = ("*const " if (const and level == 0) else "*mut ") + out
    return out


def declarations(text):
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    body = text[text.index('extern "C" {'):]
    for m in re.finditer(r"\b([A-Za-z_][\w ]*?[\s\*]+)(sage_[a-z0-9_]+)\s*\(([^;{}]*?)\)\s*;", body, flags=re.S):
        ret, name, args = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        if ret.startswith("typedef"):
            continue
        params = []
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                am = re.match(r"^(.*?)([A-Za-z_]\w*)(\[\d*\])?$", a)
                params.append((am.group(2), rust_type(am.group(1), am.group(3) is not None)))
        yield name, ret, params


def generate():
    lines = [PRELUDE]
    for name, ret, params in declarations(open(HEADER).read()):
        ps = ", ".join("%s: %s" % (("r#" + n) if n in ("type", "match", "ref", "in", "fn", "mod", "move") else n, t) for n, t in params)
        r = "" if ret == "void" else " -> " + rust_type(ret, False)
        lines.append("    pub fn %s(%s)%s;\n" % (name, ps, r))
    lines.append("}\n")
    return "".join(lines)


if __name__ == "__main__":
    src = generate()
    if "--check" in sys.argv:
        sys.exit(0 if os.path.exists(OUT) and open(OUT).read() == src else 1)
    open(OUT, "w").write(src)
    print("wrote %s (%d functions)" % (os.path.relpath(OUT), src.count("pub fn ")))
