#!/usr/bin/env python3
"""Writes src/bindings.rs from include/hs_attn.h and include/hs_kv_cache.h:  python hs-attn-sys/gen_bindings.py

The reference's bitsandbytes-sys keeps a hand-written bindings.rs and offers bindgen as an option
(crates/bitsandbytes-sys/build.rs, src/bindings.rs:15-334).  Here the extern "C" block is produced from the two headers
by this script, so that no entry point can be forgotten; structs, enums and constants are written out below by hand and
are checked against the headers by tests/test_abi.py."""
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
INC = os.path.join(HERE, "..", "include")

SCALARS = {"int": "c_int", "int32_t": "i32", "int64_t": "i64", "uint64_t": "u64", "uint8_t": "u8", "int8_t": "i8",
           "float": "f32", "size_t": "usize", "char": "c_char", "void": "c_void", "hs_stream_t": "hs_stream_t"}
OPAQUE = ["hs_cache", "hs_pool", "hs_paged_cache", "hs_compat"]
STRUCTS = ["hs_kv_layout", "hs_qk_prologue"]


def declarations(header):
    text = open(os.path.join(INC, header)).read()
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    out = []
    for m in re.finditer(r"HS_API\s+([^;{]*?)\b(hs_\w+)\s*\(([^;]*?)\)\s*;", text, flags=re.S):
        ret, name, args = " ".join(m.group(1).split()), m.group(2), " ".join(m.group(3).split())
        out.append((ret, name, [] if args in ("void", "") else [a.strip() for a in args.split(",")]))
    return out


def rust_type(c):
    """C type (without the parameter name) -> Rust."""
    c = c.strip()
    m = re.fullmatch(r"(const\s+)?(\w+)\s*((?:\*\s*(?:const\s*)?)*)", c)
    assert m, c
    const, base, stars = bool(m.group(1)), m.group(2), m.group(3)
    t = SCALARS.get(base) or (base if base in OPAQUE + STRUCTS else None)
    assert t, "unknown C type %r" % c
    ptrs = re.findall(r"\*\s*(const)?", stars)
    # innermost pointer takes the constness of the pointee; `T *const *` makes the outer pointer's pointee const
    for i, p in enumerate(ptrs):
        pointee_const = const if i == 0 else bool(ptrs[i - 1])
        t = ("*const " if pointee_const else "*mut ") + t
    return t


def split_param(p):
    m = re.fullmatch(r"(.*?)(\w+)\s*(\[\d*\])?", p.strip())
    ctype, name, arr = m.group(1).strip(), m.group(2), m.group(3)
    if arr:
        ctype += " *"
    name = name.lower()
    if name in ("type", "ref", "in", "fn", "mod"):
        name += "_"
    return ctype, name


def extern_block(header):
    lines = []
    for ret, name, params in declarations(header):
        ps = ", ".join("%s: %s" % (n, rust_type(t)) for t, n in map(split_param, params))
        r = "" if ret == "void" else " -> " + rust_type(ret)
        lines.append("    pub fn %s(%s)%s;" % (name, ps, r))
    return "\n".join(lines)


HEAD = '''//! Raw bindings of libhs_attn.so (include/hs_attn.h) and libhs_kv_cache.so (include/hs_kv_cache.h).
//! The `extern "C"` blocks are generated by gen_bindings.py from the headers; do not edit them by hand.
#![allow(non_camel_case_types)]
use std::ffi::{c_char, c_int, c_void};

/// `hipStream_t`; null = the default stream (what tch / libtorch uses), as `bnb_stream_t`.
pub type hs_stream_t = *mut c_void;

pub const HS_ATTN_ABI_VERSION: c_int = @ABI@;
pub const HS_ATTN_ABI_REVISION: c_int = @REVISION@;

// enum hs_status
pub const HS_OK: c_int = 0;
pub const HS_ERR_INVALID_ARGUMENT: c_int = 1;
pub const HS_ERR_OVERFLOW: c_int = 2;
pub const HS_ERR_WORKSPACE: c_int = 3;
pub const HS_ERR_LAUNCH: c_int = 4;
pub const HS_ERR_POOL_EXHAUSTED: c_int = 5;
pub const HS_ERR_BUSY: c_int = 6;
// enum hs_dtype
pub const HS_BF16: c_int = 0;
pub const HS_F32: c_int = 1;
pub const HS_F16: c_int = 2;
// enum hs_qk_norm_kind
pub const HS_QKNORM_NONE: c_int = 0;
pub const HS_QKNORM_LLAMA: c_int = 1;
pub const HS_QKNORM_QWEN35: c_int = 2;
// enum hs_kv_quant (storage format of a cache object)
pub const HS_KV_NONE: c_int = 0;
pub const HS_KV_INT8: c_int = 1;
pub const HS_KV_FP8: c_int = 2;
// enum hs_kv_quant_mode (KvQuantMode of the compatibility fingerprint)
pub const HS_KVQ_NONE: c_int = 0;
pub const HS_KVQ_INT8: c_int = 1;
pub const HS_KVQ_NF4: c_int = 2;
pub const HS_KVQ_FP4: c_int = 3;
pub const HS_KVQ_INT8_TOKEN: c_int = 4;
pub const HS_KVQ_FP8_E4M3FN_HEAD: c_int = 5;
// enum hs_cache_reuse
pub const HS_REUSE: c_int = 0;
pub const HS_STAMP_FRESH: c_int = 1;
pub const HS_DISCARD_AND_RECOMPUTE: c_int = 2;

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct hs_kv_layout {
    pub code_stride_seq: i64,
    pub code_stride_head: i64,
    pub scale_stride_seq: i64,
    pub scale_stride_head: i64,
    pub capacity_tokens: i32,
    pub block_table_stride: i32,
    pub k_block_table: *const i32,
    pub v_block_table: *const i32,
    pub total_tokens_hint: i64,
    pub prefill_columns_hint: i32,
    pub prefill_window: i32,
    pub out_gate: *const c_void,
    pub prefill_q_prologue: *const hs_qk_prologue,
    pub prefill_split_workspace: *mut c_void,
    pub prefill_split_workspace_bytes: i64,
    pub prefill_key_splits: i32,
    pub attn_sinks: i32,
    pub prefill_shadow: *mut c_void,
    pub prefill_shadow_bytes: i64,
    pub prefill_shadow_tokens: i32,
    pub decode_window: i32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct hs_qk_prologue {
    pub norm_kind: i32,
    pub norm_eps: f32,
    pub q_norm_weight: *const c_void,
    pub k_norm_weight: *const c_void,
    pub q_norm_head_stride: i32,
    pub k_norm_head_stride: i32,
    pub rope_sin: *const c_void,
    pub rope_cos: *const c_void,
    pub rope_len: i32,
    pub rotary_dim: i32,
}

#[repr(C)] pub struct hs_cache { _private: [u8; 0] }
#[repr(C)] pub struct hs_pool { _private: [u8; 0] }
#[repr(C)] pub struct hs_paged_cache { _private: [u8; 0] }
#[repr(C)] pub struct hs_compat { _private: [u8; 0] }
'''


def main():
    header = open(os.path.join(HERE, "..", "include", "hs_attn.h")).read()
    out = HEAD
    for mark, name in (("@ABI@", "HS_ATTN_ABI_VERSION"), ("@REVISION@", "HS_ATTN_ABI_REVISION")):
        number = re.search(r"#define\s+%s\s+(\d+)" % name, header).group(1)
        out = out.replace(mark, number)
    out += '\n// ---- include/hs_attn.h -> libhs_attn.so\n#[link(name = "hs_attn")]\nextern "C" {\n%s\n}\n' % extern_block("hs_attn.h")
    out += ('\n// ---- include/hs_kv_cache.h -> libhs_kv_cache.so (optional host mirror)\n#[cfg(feature = "kv-cache")]\n'
            '#[link(name = "hs_kv_cache")]\nextern "C" {\n%s\n}\n' % extern_block("hs_kv_cache.h"))
    path = os.path.join(HERE, "src", "bindings.rs")
    open(path, "w").write(out)
    print(path, len(declarations("hs_attn.h")), "+", len(declarations("hs_kv_cache.h")), "functions")


if __name__ == "__main__":
    main()
