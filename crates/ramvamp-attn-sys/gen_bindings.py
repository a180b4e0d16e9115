#!/usr/bin/env python3
"""Generates this crate's src/lib.rs and build.rs from the library itself:

    python crates/ramvamp-attn-sys/gen_bindings.py          # rewrite both
    python crates/ramvamp-attn-sys/gen_bindings.py --check  # exit 1 if stale

src/lib.rs declares, one to one, every constant, struct and function of
include/*.h (the C ABI of libramvamp_attn.so); build.rs compiles exactly the
sources, with exactly the flags, that ramvamp_amd/build.py compiles. The
headers use a small, regular subset of C (fixed-width integers, size_t,
float/double, pointers to those or to the ABI's own structs, #define'd
integer constants), which is all this translator handles; anything else is
an error, not a guess.
"""
from __future__ import annotations

import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
INCLUDE = os.path.join(ROOT, "include")
HEADERS = ["ramvamp_attn.h", "ramvamp_gemv.h", "ramvamp_block.h", "ramvamp_router.h", "ramvamp_paged.h",
           "ramvamp_floors.h"]

SCALARS = {"void": "()", "int": "c_int", "char": "c_char", "float": "f32", "double": "f64", "size_t": "usize",
           "int8_t": "i8", "uint8_t": "u8", "int16_t": "i16", "uint16_t": "u16", "int32_t": "i32",
           "uint32_t": "u32", "int64_t": "i64", "uint64_t": "u64"}


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", " ", text, flags=re.S)


def rust_type(ctype: str, known: set[str]) -> str:
    """`const float*` -> `*const f32`, `rv_kv**` -> `*mut *mut rv_kv`, ..."""
    t = " ".join(ctype.replace("*", " * ").split())
    stars = t.count("*")
    base = t.replace("*", "").strip()
    const = base.startswith("const ")
    base = base.replace("const ", "").strip()
    if base in SCALARS:
        r = "c_void" if (base == "void" and stars) else SCALARS[base]
    elif base in known:
        r = base
    else:
        raise ValueError(f"unsupported C type {ctype!r}")
    for i in range(stars):
        r = ("*const " if (const and i == 0) else "*mut ") + r
    return r


def parse(headers: list[str]):
    consts, structs, funcs, opaque, enums = [], [], [], [], []
    for h in headers:
        raw = open(os.path.join(INCLUDE, h)).read()
        for m in re.finditer(r"^#define\s+(RV_[A-Z0-9_]+)\s+(.+?)\s*(?:/\*.*)?$", raw, flags=re.M):
            name, val = m.group(1), m.group(2).strip()
            if name.endswith("_H"):
                continue
            if val.startswith("((size_t)"):
                consts.append((name, "usize", val.replace("((size_t)", "(").replace("((", "(")))
            elif val.endswith("u"):
                consts.append((name, "u32", val[:-1]))
            else:
                consts.append((name, "i32", val))
        text = strip_comments(raw)
        text = re.sub(r"^\s*#.*$", "", text, flags=re.M)
        text = text.replace('extern "C" {', "").replace("extern \"C\"", "")
        for m in re.finditer(r"typedef\s+struct\s+(\w+)\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
            fields = []
            for f in m.group(2).split(";"):
                f = " ".join(f.split())
                if not f:
                    continue
                parts = [x.strip() for x in f.split(",")]  # `uint64_t a, b, c` declares several
                fm = re.match(r"(.+?)\s*(\w+)\s*(?:\[(\d+)\])?$", parts[0])
                ftype = fm.group(1)
                fields.append((fm.group(2), ftype, fm.group(3)))
                for extra_decl in parts[1:]:
                    em = re.match(r"(\w+)\s*(?:\[(\d+)\])?$", extra_decl)
                    fields.append((em.group(1), ftype, em.group(2)))
            structs.append((m.group(3), fields))
        for m in re.finditer(r"typedef\s+enum\s+(\w+)\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
            enums.append(m.group(3))
            for item in m.group(2).split(","):
                k, v = [x.strip() for x in item.split("=")]
                consts.append((k, "i32", v))
        for m in re.finditer(r"typedef\s+struct\s+(\w+)\s+(\w+)\s*;", text):
            opaque.append(m.group(2))
        body = re.sub(r"typedef\s+(struct|enum)\s+\w+\s*\{.*?\}\s*\w+\s*;", "", text, flags=re.S)
        body = re.sub(r"typedef\s+struct\s+\w+\s+\w+\s*;", "", body)
        for m in re.finditer(r"([A-Za-z_][\w\s\*]*?)\b(rv_\w+)\s*\(([^;{]*?)\)\s*;", body, flags=re.S):
            ret, name, params = " ".join(m.group(1).split()), m.group(2), " ".join(m.group(3).split())
            plist = []
            if params and params != "void":
                for p in params.split(","):
                    pm = re.match(r"(.+?)\s*(\w+)$", p.strip())
                    plist.append((pm.group(2), pm.group(1)))
            funcs.append((name, ret, plist))
    return consts, structs, funcs, opaque, enums


def gen_lib_rs() -> str:
    consts, structs, funcs, opaque, enums = parse(HEADERS)
    known = set(opaque) | {s for s, _ in structs} | set(enums)
    out = ["// Generated by gen_bindings.py from include/*.h; do not edit by hand.",
           "//! Raw bindings to libramvamp_attn (the MI355X attention hot path's C ABI):",
           "//! one declaration per symbol of include/ramvamp_attn.h, ramvamp_gemv.h,",
           "//! ramvamp_block.h, ramvamp_router.h, ramvamp_paged.h and ramvamp_floors.h. The safe wrapper",
           "//! that keeps the reference's signatures is crates/ramvamp-attn.",
           "#![allow(non_camel_case_types, clippy::missing_safety_doc)]",
           "use std::os::raw::{c_char, c_int, c_void};", ""]
    for name, ty, val in consts:
        out.append(f"pub const {name}: {ty} = {val};")
    out.append("")
    for e in enums:
        out.append(f"pub type {e} = i32;")
    for o in opaque:
        out.append(f"#[repr(C)]\npub struct {o} {{\n    _private: [u8; 0],\n}}")
    for name, fields in structs:
        derive = "#[derive(Clone, Copy)]"
        body = []
        for fname, ftype, arr in fields:
            rt = rust_type(ftype, known)
            body.append(f"    pub {fname}: [{rt}; {arr}]," if arr else f"    pub {fname}: {rt},")
        out.append(f"#[repr(C)]\n{derive}\npub struct {name} {{\n" + "\n".join(body) + "\n}")
    out.append("")
    out.append('extern "C" {')
    for name, ret, plist in funcs:
        args = ", ".join(f"{p}: {rust_type(t, known)}" for p, t in plist)
        rt = rust_type(ret, known)
        out.append(f"    pub fn {name}({args})" + ("" if rt == "()" else f" -> {rt}") + ";")
    out.append("}")
    return "\n".join(out) + "\n"


def gen_build_rs() -> str:
    sys.path.insert(0, ROOT)
    from ramvamp_amd import build as B  # the library's own build recipe: sources, flags, per-source extras

    srcs = ",\n".join(f'        "{s}"' for s in B.SOURCES)
    flags = ", ".join(f'"{f}"' for f in B.FLAGS)
    extra = ",\n".join(f'        ("{s}", &[{", ".join(repr(x).replace(chr(39), chr(34)) for x in v)}])'
                       for s, v in B.EXTRA.items())
    return f'''// Generated by gen_bindings.py from ramvamp_amd/build.py; do not edit by hand.
// Compiles the HIP sources for gfx950 with hipcc (no cmake, no CUDA, no other
// backend) into OUT_DIR/libramvamp_attn.so and links it. RAMVAMP_AMD_DIR
// points at the repository that holds ramvamp_amd/csrc and include/.
use std::{{env, path::PathBuf, process::Command}};

const SOURCES: &[&str] = &[
{srcs},
];
const FLAGS: &[&str] = &[{flags}];
const EXTRA: &[(&str, &[&str])] = &[
{extra},
];

fn main() {{
    let root = PathBuf::from(env::var("RAMVAMP_AMD_DIR").unwrap_or_else(|_| "../..".into()));
    let csrc = root.join("ramvamp_amd/csrc");
    let out = PathBuf::from(env::var("OUT_DIR").unwrap());
    let hipcc = env::var("HIPCC").unwrap_or_else(|_| "/opt/rocm/bin/hipcc".into());
    let mut objs = Vec::new();
    for src in SOURCES {{
        let obj = out.join(format!("{{src}}.o"));
        let mut cmd = Command::new(&hipcc);
        cmd.args(FLAGS);
        if let Some((_, more)) = EXTRA.iter().find(|(s, _)| s == src) {{
            cmd.args(*more);
        }}
        let status = cmd.arg("-c").arg("-o").arg(&obj).arg(csrc.join(src)).status().expect("hipcc");
        assert!(status.success(), "hipcc failed on {{src}}");
        objs.push(obj);
    }}
    let status = Command::new(&hipcc)
        .args(["--offload-arch=gfx950", "-shared", "-fPIC", "-o"])
        .arg(out.join("libramvamp_attn.so"))
        .args(&objs)
        .status()
        .expect("hipcc link");
    assert!(status.success(), "hipcc link failed");
    println!("cargo:rustc-link-search=native={{}}", out.display());
    println!("cargo:rustc-link-lib=dylib=ramvamp_attn");
    println!("cargo:rerun-if-changed={{}}", csrc.display());
    println!("cargo:rerun-if-changed={{}}", root.join("include").display());
}}
'''


def main() -> int:
    targets = {os.path.join(HERE, "src", "lib.rs"): gen_lib_rs(), os.path.join(HERE, "build.rs"): gen_build_rs()}
    if "--check" in sys.argv:
        stale = [p for p, text in targets.items() if not os.path.exists(p) or open(p).read() != text]
        for p in stale:
            print(f"stale: {os.path.relpath(p, ROOT)} (run gen_bindings.py)", file=sys.stderr)
        return 1 if stale else 0
    for p, text in targets.items():
        os.makedirs(os.path.dirname(p), exist_ok=True)
        with open(p, "w") as f:
            f.write(text)
    return 0


if __name__ == "__main__":
    sys.exit(main())
