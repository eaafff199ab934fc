"""Writes rust/autograph-b200-sys/src/lib.rs from include/autograph_b200.h, so that the Rust
declarations cannot drift from the C ABI (tests/test_abi.py compares the two symbol sets).

    python rust/gen_sys.py
"""
from __future__ import annotations

import re
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "autograph_b200.h"
OUT = ROOT / "rust" / "autograph-b200-sys" / "src" / "lib.rs"

TYPES = {
    "int": "c_int", "int32_t": "i32", "int64_t": "i64", "uint64_t": "u64", "uint8_t": "u8",
    "uint32_t": "u32", "size_t": "usize", "float": "f32", "double": "f64", "void": "c_void",
    "char": "c_char", "ag_dtype": "c_int", "ag_device": "ag_device", "ag_model": "ag_model",
    "ag_comm": "ag_comm", "ag_conv2_options": "ag_conv2_options", "ag_conv_stage": "ag_conv_stage",
    "ag_layer_spec": "ag_layer_spec", "ag_polar_matrix": "ag_polar_matrix", "ag_muon_matrix": "ag_muon_matrix",
}


def rust_type(c: str) -> str:
    c = c.strip()
    const = False
    stars = c.count("*")
    base = c.replace("*", " ").replace("const", " ")
    const = "const" in c.split("*")[0]
    base = base.split()[0] if base.split() else "void"
    t = TYPES[base]
    # C reads declarators right to left; every level here is either `const T *` or `T *`,
    # and a trailing `*const` level only guards the pointer itself
    levels = [seg for seg in c.split("*")]
    for i in range(stars):
        inner_const = "const" in levels[i] if i < len(levels) else False
        t = f"*{'const' if inner_const else 'mut'} {t}"
    return t


def parse():
    text = HEADER.read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    funcs = []
    for m in re.finditer(r"AG_API\s+([\w\s\*]+?)\b(ag_\w+)\s*\(([^;]*?)\)\s*;", text, flags=re.S):
        ret, name, args = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        params = []
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                pm = re.match(r"(.*?)(\w+)$", a)
                ctype, pname = pm.group(1).strip(), pm.group(2)
                params.append((pname, rust_type(ctype)))
        funcs.append((name, params, None if ret == "int" and False else rust_type(ret)))
    return funcs


def main():
    funcs = parse()
    lines = [
        "//! Raw bindings of `libautograph_b200.so` (include/autograph_b200.h), generated by",
        "//! rust/gen_sys.py.  NOT COMPILED where this repository is developed (no Rust toolchain on",
        "//! those machines): it is the crate a maintainer of autograph would add behind a `b200`",
        "//! cargo feature.  Every function returns an ag_status (0 = ok); `check` turns it into the",
        "//! `anyhow::Result` the reference uses everywhere.",
        "#![allow(non_camel_case_types)]",
        "use std::os::raw::{c_char, c_int, c_void};",
        "",
        "#[repr(C)] pub struct ag_device { _private: [u8; 0] }",
        "#[repr(C)] pub struct ag_model { _private: [u8; 0] }",
        "#[repr(C)] pub struct ag_comm { _private: [u8; 0] }",
        "",
        "pub const AG_F32: c_int = 0;",
        "pub const AG_BF16: c_int = 1;",
        "pub const AG_U8: c_int = 2;",
        "pub const AG_U16: c_int = 3;",
        "pub const AG_U32: c_int = 4;",
        "",
        "pub const AG_OK: c_int = 0;",
        "pub const AG_ERR_INVALID: c_int = -1;",
        "pub const AG_ERR_SHAPE: c_int = -2;",
        "pub const AG_ERR_DTYPE: c_int = -3;",
        "pub const AG_ERR_CUDA: c_int = -4;",
        "pub const AG_ERR_OOM: c_int = -5;",
        "pub const AG_ERR_DEVICE_TIMEOUT: c_int = -6;",
        "pub const AG_ERR_UNSUPPORTED: c_int = -7;",
        "pub const AG_ERR_LIMIT: c_int = -8;",
        "",
        "#[repr(C)]",
        "#[derive(Clone, Copy, Debug, Default)]",
        "pub struct ag_conv2_options {",
        "    pub filter: [i32; 2],",
        "    pub padding: [i32; 2],",
        "    pub stride: [i32; 2],",
        "    pub dilation: [i32; 2],",
        "}",
        "",
        "#[repr(C)]",
        "#[derive(Clone, Copy)]",
        "pub struct ag_conv_stage {",
        "    pub w: *const c_void,",
        "    pub bias: *const c_void,",
        "    pub oc: i64,",
        "    pub options: ag_conv2_options,",
        "    pub relu: i32,",
        "    pub pool: [i32; 2],",
        "}",
        "",
        "#[repr(C)]",
        "#[derive(Clone, Copy, Debug, Default)]",
        "pub struct ag_layer_spec {",
        "    pub kind: i32,",
        "    pub a: i32,",
        "    pub b: i32,",
        "    pub c: i32,",
        "    pub d: i32,",
        "    pub bias: i32,",
        "}",
        "",
        "#[repr(C)]",
        "#[derive(Clone, Copy)]",
        "pub struct ag_polar_matrix {",
        "    pub g: *const c_void,",
        "    pub o: *mut c_void,",
        "    pub rows: i64,",
        "    pub cols: i64,",
        "}",
        "",
        "#[repr(C)]",
        "#[derive(Clone, Copy)]",
        "pub struct ag_muon_matrix {",
        "    pub w: *mut c_void,",
        "    pub g: *const c_void,",
        "    pub v: *mut f32,",
        "    pub rows: i64,",
        "    pub cols: i64,",
        "    pub scale: f32,",
        "}",
        "",
        '#[link(name = "autograph_b200")]',
        'extern "C" {',
    ]
    for name, params, ret in funcs:
        args = ", ".join(f"{'r#' + p if p in ('in', 'type', 'box') else p}: {t}" for p, t in params)
        lines.append(f"    pub fn {name}({args}) -> {ret};")
    lines += [
        "}",
        "",
        "/// status -> anyhow::Error with the library's message (the reference returns",
        "/// `anyhow::Result` everywhere and `bail!`s on shape and type mismatches).",
        "pub fn check(status: c_int) -> anyhow::Result<()> {",
        "    if status == AG_OK {",
        "        return Ok(());",
        "    }",
        "    let msg = unsafe { std::ffi::CStr::from_ptr(ag_last_error()) }.to_string_lossy().into_owned();",
        '    Err(anyhow::anyhow!("autograph_b200 ({status}): {msg}"))',
        "}",
        "",
    ]
    OUT.write_text("\n".join(lines))
    print(OUT, len(funcs), "functions")


if __name__ == "__main__":
    main()
