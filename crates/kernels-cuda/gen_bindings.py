#!/usr/bin/env python
"""Writes src/ffi.rs and src/dispatch.rs from include/runit_cuda.h and include/runit_gguf.h.

ffi.rs declares EVERY function of the two headers; dispatch.rs wraps every operator (first argument a context, int32
status) as a free function with the reference's shape, `op(ctx: &CudaContext, buffers: &DeviceBuffer..., dims...) ->
Result<()>` (crates/kernels/src/dispatch.rs).  Run from anywhere: `python crates/kernels-cuda/gen_bindings.py`;
tests/test_cabi.py checks that the committed files are what this script writes."""
import re
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent.parent
HEADERS = [ROOT / "include" / "runit_cuda.h", ROOT / "include" / "runit_gguf.h"]

SCALARS = {"int32_t": "i32", "uint32_t": "u32", "uint64_t": "u64", "int64_t": "i64", "size_t": "usize", "float": "f32"}
OPAQUE = ["runit_ctx_t", "runit_graph_t", "runit_model_t", "runit_gguf_t"]
STRUCTS = ["runit_model_cfg", "runit_model_weights", "runit_sampler_cfg", "runit_gguf_tensor_info",
           "runit_layer_desc", "runit_layered_cfg", "runit_layered_weights", "runit_latent_cfg",
           "runit_heads_cfg", "runit_retention_cfg", "runit_ssm_cfg", "runit_linear_cfg", "runit_paged_cfg", "runit_paged_batch"]
# operators that are not GPU ops of the dispatch layer (context, buffers, recording): wrapped by hand in context.rs
NOT_OPS = {"runit_ctx_create", "runit_ctx_create_on_stream", "runit_ctx_destroy", "runit_flush", "runit_buf_alloc", "runit_buf_free",
           "runit_memcpy_h2d", "runit_memcpy_d2h", "runit_memset", "runit_set_tuning", "runit_graph_begin", "runit_graph_end",
           "runit_graph_launch", "runit_graph_destroy", "runit_model_create", "runit_model_create_ep", "runit_model_create_layered"}


def parse(path):
    text = re.sub(r"/\*.*?\*/", " ", path.read_text(), flags=re.S)
    text = re.sub(r"//[^\n]*", " ", text)
    out = []
    for m in re.finditer(r"([A-Za-z_][\w\s\*]*?)\b(runit_\w+)\s*\(([^;{()]*)\)\s*;", text):
        ret = " ".join(m.group(1).split()).replace(" *", "*")
        if ret.startswith("typedef") or "(" in ret:
            continue
        args = []
        raw = m.group(3).strip()
        if raw and raw != "void":
            for i, a in enumerate(raw.split(",")):
                a = " ".join(a.split())
                a = re.sub(r"\s*\*\s*", "* ", a).replace("* *", "**").strip()
                parts = a.split(" ")
                name = "a%d" % i
                if len(parts) > 1 and not parts[-1].endswith("*") and parts[-1] not in SCALARS and parts[-1] not in ("void", "char"):
                    name, parts = parts[-1], parts[:-1]
                args.append((" ".join(parts).replace(" *", "*").replace("* const*", "* const*"), name))
        out.append((ret, m.group(2), args))
    return out


def rust_type(c):
    c = c.strip()
    if c in SCALARS:
        return SCALARS[c]
    if c in ("const void*", "void*"):
        return "*const c_void" if c.startswith("const") else "*mut c_void"
    if c == "const char*":
        return "*const c_char"
    if c in ("void* const*", "const void* const*"):
        return "*const *mut c_void"
    if c == "void**":
        return "*mut *mut c_void"
    m = re.fullmatch(r"(const )?(\w+)(\*+)", c)
    if m:
        base = m.group(2)
        inner = SCALARS.get(base, base)
        ptr = "*const " if m.group(1) else "*mut "
        t = inner
        for _ in m.group(3):
            t = ptr + t
        return t
    raise SystemExit("no Rust type for %r" % c)


def rust_name(n):
    return "r#" + n if n in ("type", "ref", "in", "fn", "loop", "match", "move") else n


def gen():
    fns = [f for h in HEADERS for f in parse(h)]
    ffi = ["//! `extern \"C\"` declarations of every function in include/runit_cuda.h and include/runit_gguf.h.",
           "//! Generated by gen_bindings.py; do not edit.", "#![allow(non_camel_case_types)]", "use std::ffi::c_void;",
           "use std::os::raw::c_char;", ""]
    for o in OPAQUE:
        ffi += ["#[repr(C)]", "pub struct %s {" % o, "    _private: [u8; 0],", "}"]
    ffi += ["", "/// Field for field the C structs of the headers.", "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_model_cfg {",
            "    pub n_layers: i32, pub hidden: i32, pub n_heads: i32, pub n_kv_heads: i32, pub head_dim: i32, pub vocab: i32,",
            "    pub n_experts: i32, pub top_k: i32, pub ff: i32, pub max_seq: i32, pub renorm: i32,", "    pub eps: f32, pub theta: f32,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_model_weights {",
            "    pub tok_emb: *const c_void, pub attn_norm: *const c_void, pub ffn_norm: *const c_void, pub out_norm: *const c_void,",
            "    pub wq: *const c_void, pub wk: *const c_void, pub wv: *const c_void, pub wo: *const c_void, pub router: *const c_void,",
            "    pub gate: *const c_void, pub up: *const c_void, pub down: *const c_void, pub lm_head: *const c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_sampler_cfg {",
            "    pub temperature: f32, pub top_k: i32, pub top_p: f32, pub repetition_penalty: f32, pub min_tokens: i32,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_gguf_tensor_info {",
            "    pub name: *const c_char, pub dtype: u32, pub n_dims: u32, pub ne: [u64; 4],",
            "    pub data_offset: u64, pub num_elements: u64, pub data_size: u64,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_layer_desc {",
            "    pub heads: i32, pub dim: i32, pub rot_dim: i32, pub vdim: i32, pub kv_rank: i32, pub kv_from: i32,",
            "    pub scale: f32, pub rot_base: f32,",
            "    pub ff_kind: i32, pub ff_act: i32, pub ff: i32, pub n_experts: i32, pub top_k: i32, pub score: i32, pub renorm: i32, pub shared_ff: i32,",
            "    pub norm1: *const c_void, pub norm2: *const c_void, pub w_q: *const c_void, pub kv_norm: *const c_void,",
            "    pub w_ukv: *const c_void, pub w_o: *const c_void, pub ff_up: *const c_void, pub ff_down: *const c_void,",
            "    pub router: *const c_void, pub shared_up: *const c_void, pub shared_down: *const c_void,",
            "    pub mixer: i32, pub at_heads: i32, pub at_kv_heads: i32, pub at_dim: i32, pub at_vdim: i32, pub at_window: i32, pub at_unit_qk: i32,",
            "    pub rt_heads: i32, pub rt_dim: i32, pub rt_vdim: i32, pub rt_rot_dims: i32,",
            "    pub ss_heads: i32, pub ss_vdim: i32, pub ss_state: i32, pub ss_groups: i32, pub ss_taps: i32, pub ss_norm_groups: i32,",
            "    pub at_scale: f32, pub at_out_scale: f32, pub rt_rot_base: f32, pub rt_out_scale: f32,",
            "    pub at_slopes: *const c_void, pub rt_decay: *const c_void, pub ss_conv: *const c_void, pub ss_conv_b: *const c_void,",
            "    pub ss_dt_bias: *const c_void, pub ss_a: *const c_void, pub ss_skip: *const c_void, pub ss_norm: *const c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_latent_cfg {",
            "    pub heads: u32, pub dim: u32, pub rot_dim: u32, pub vdim: u32, pub kv_rank: u32,", "    pub scale: f32, pub eps: f32,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_heads_cfg {",
            "    pub heads: u32, pub kv_heads: u32, pub dim: u32, pub vdim: u32, pub window: u32, pub cap: u32, pub unit_qk: u32,",
            "    pub scale: f32, pub out_scale: f32, pub eps: f32,",
            "    pub slopes: *const c_void, pub k_cache: *mut c_void, pub v_cache: *mut c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_retention_cfg {",
            "    pub heads: u32, pub dim: u32, pub vdim: u32, pub rot_dims: u32, pub out_scale: f32,",
            "    pub freq: *const c_void, pub decay: *const c_void, pub state: *mut c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_ssm_cfg {",
            "    pub heads: u32, pub vdim: u32, pub state_dim: u32, pub groups: u32, pub taps: u32,",
            "    pub conv: *const c_void, pub conv_b: *const c_void, pub dt_bias: *const c_void, pub a: *const c_void, pub skip: *const c_void,",
            "    pub state: *mut c_void, pub ring: *mut c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_linear_cfg {",
            "    pub heads: u32, pub groups: u32, pub dk: u32, pub dv: u32, pub ldq: u32, pub ldk: u32, pub ldv: u32, pub ldo: u32,",
            "    pub q: *const c_void, pub k: *const c_void, pub v: *const c_void, pub dt: *const c_void, pub log_decay: *const c_void,",
            "    pub decay: *const c_void, pub skip: *const c_void, pub state: *mut c_void, pub out: *mut c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_paged_cfg {",
            "    pub heads: u32, pub kv_heads: u32, pub dim: u32, pub page: u32, pub n_pages: u32, pub type_: i32, pub window: u32,",
            "    pub scale: f32, pub cap: f32, pub slopes: *const c_void, pub k_pages: *mut c_void, pub v_pages: *mut c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_paged_batch {",
            "    pub n_seqs: u32, pub rows: u32, pub table_ld: u32, pub shared_len: u32,",
            "    pub table: *const c_void, pub q_start: *const c_void, pub kv_len: *const c_void,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_layered_cfg {",
            "    pub n_layers: i32, pub width: i32, pub vocab: i32, pub max_seq: i32, pub exact: i32, pub post_norm: i32,",
            "    pub eps: f32, pub embed_scale: f32, pub logit_cap: f32,", "}",
            "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", "pub struct runit_layered_weights {",
            "    pub embed: *const c_void, pub embed_norm: *const c_void, pub final_norm: *const c_void, pub head: *const c_void,", "}", ""]
    ffi += ["pub const RUNIT_OK: i32 = 0;", "pub const RUNIT_ERR_NO_DEVICE: i32 = 1;", "pub const RUNIT_ERR_BAD_ARG: i32 = 2;",
            "pub const RUNIT_ERR_BUFFER_SIZE: i32 = 3;", "pub const RUNIT_ERR_LAUNCH: i32 = 4;", "pub const RUNIT_ERR_NCCL: i32 = 5;",
            "pub const RUNIT_ERR_TIMEOUT: i32 = 6;", "pub const RUNIT_ERR_UNSUPPORTED: i32 = 7;", "pub const RUNIT_ERR_ALLOC: i32 = 8;",
            "pub const RUNIT_BUF_DEVICE: i32 = 0;", "pub const RUNIT_BUF_HOST_VISIBLE: i32 = 1;", "", "extern \"C\" {"]
    for ret, name, args in fns:
        a = ", ".join("%s: %s" % (rust_name(n), rust_type(t)) for t, n in args)
        r = "" if ret == "void" else " -> " + rust_type(ret)
        ffi.append("    pub fn %s(%s)%s;" % (name, a, r))
    ffi += ["}", ""]
    (HERE / "src" / "ffi.rs").write_text("\n".join(ffi))

    d = ["//! The free functions of crates/kernels/src/dispatch.rs for the quantized decode path (same names, same argument",
         "//! order), plus the operators that have no twin there, forwarding to librunit_cuda.so.  `ctx: &MetalContext` becomes",
         "//! `&CudaContext`, `&metal::Buffer` becomes `&DeviceBuffer`, tables of peer pointers are slices of raw device pointers.",
         "//! Generated by gen_bindings.py from include/runit_cuda.h (which cites the dispatch.rs line of every twin); do not edit.",
         "#![allow(clippy::too_many_arguments)]", "use std::ffi::c_void;", "", "use crate::context::{CudaContext, DeviceBuffer};",
         "use crate::error::Result;", "use crate::ffi;", "", "type B = DeviceBuffer;", ""]
    for ret, name, args in fns:
        if ret != "int32_t" or not args or args[0][0] != "runit_ctx_t*" or name in NOT_OPS:
            continue
        params, call = ["ctx: &CudaContext"], ["ctx.raw"]
        ok = True
        for t, n in args[1:]:
            n = rust_name(n)
            if t == "const void*":
                params.append("%s: &B" % n); call.append("%s.ptr as *const c_void" % n)
            elif t == "void*":
                params.append("%s: &B" % n); call.append("%s.ptr" % n)
            elif t in ("void* const*", "const void* const*"):
                params.append("%s: &[*mut c_void]" % n); call.append("%s.as_ptr()" % n)
            elif t in SCALARS:
                params.append("%s: %s" % (n, SCALARS[t])); call.append(n)
            else:
                ok = False
        if not ok:
            continue
        short = name[len("runit_"):]
        d.append("pub fn %s(%s) -> Result<()> {" % (short, ", ".join(params)))
        d.append("    ctx.check(unsafe { ffi::%s(%s) })" % (name, ", ".join(call)))
        d.append("}")
    d += ["", "/// Launch-shape variants the engine selects by row count (`use_mr = m >= 128`, crates/engine/src/forward.rs:134,193)",
          "/// are the same kernel here; the names exist so that WeightBuf compiles unchanged.", ""]
    (HERE / "src" / "dispatch.rs").write_text("\n".join(d))
    return fns


if __name__ == "__main__":
    fns = gen()
    print("wrote ffi.rs (%d functions) and dispatch.rs" % len(fns))
