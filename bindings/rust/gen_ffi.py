#!/usr/bin/env python3
"""Generate bindings/rust/src/ffi.rs (the `extern "C"` block a Rust host links against) from
include/paged_infer_cuda.h, so that the Rust side can never drift from the C ABI.

    python bindings/rust/gen_ffi.py            # rewrite src/ffi.rs
    python bindings/rust/gen_ffi.py --check    # exit 1 if src/ffi.rs is out of date

The output cannot be compiled in this repository's environment (no rustc); it is plain generated text."""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "paged_infer_cuda.h")
OUT = os.path.join(HERE, "src", "ffi.rs")

SCALARS = {"int": "i32", "int32_t": "i32", "uint32_t": "u32", "int8_t": "i8", "uint16_t": "u16", "uint64_t": "u64", "int64_t": "i64", "size_t": "usize",
           "float": "f32", "double": "f64", "char": "std::ffi::c_char", "void": "std::ffi::c_void", "pi_status": "i32", "pi_split": "i32"}
OPAQUE = ["pi_ctx", "pi_linear", "pi_kv_pool", "pi_model", "pi_state_pool", "pi_kv8_pool"]


def rust_name(c: str) -> str:
    return "".join(p.capitalize() for p in c.split("_"))


def rust_type(c: str) -> str:
    c = c.strip()
    ptr = c.count("*")
    base = c.replace("*", " ").split()
    const = "const" in base
    base = [b for b in base if b not in ("const", "struct")]
    name = " ".join(base)
    t = SCALARS.get(name) or (rust_name(name) if name.startswith("pi_") else None)
    if t is None:
        raise SystemExit(f"unknown C type {c!r}")
    for _ in range(ptr):
        t = ("*const " if const else "*mut ") + t
        const = False          # only the innermost level of the C declarations here is const-qualified
    return t


def split_decl(decl: str):
    """'const float* x_dev' -> ('const float*', 'x_dev')"""
    decl = re.sub(r"/\*.*?\*/", "", decl).strip()
    m = re.match(r"^(.*?)([A-Za-z_][A-Za-z0-9_]*)$", decl)
    return m.group(1).strip(), m.group(2)


def generate() -> str:
    text = open(HEADER).read()
    code = re.sub(r"/\*.*?\*/", lambda m: " " * 0, text, flags=re.S)
    out = ["// GENERATED by bindings/rust/gen_ffi.py from include/paged_infer_cuda.h - do not edit.",
           "#![allow(non_camel_case_types, dead_code)]", ""]
    for m in re.finditer(r"enum\s*\{([^}]*)\}\s*\w*\s*;", code):
        for item in m.group(1).split(","):
            if "=" in item:
                k, v = [s.strip() for s in item.split("=")]
                out.append(f"pub const {k}: i32 = {v};")
    for m in re.finditer(r"#define\s+(PI_[A-Z0-9_]+)\s+(-?\d+)", code):
        out.append(f"pub const {m.group(1)}: i32 = {m.group(2)};")
    out.append("")
    for name in OPAQUE:
        out.append(f"#[repr(C)] pub struct {rust_name(name)} {{ _private: [u8; 0] }}")
    out.append("")
    for m in re.finditer(r"typedef\s+struct\s*\{(.*?)\}\s*(pi_[a-z0-9_]+)\s*;", code, flags=re.S):
        fields = []
        for stmt in m.group(1).split(";"):
            stmt = stmt.strip()
            if not stmt:
                continue
            first_type, first_name = split_decl(stmt.split(",")[0])
            fields.append((first_name, rust_type(first_type)))
            for extra in stmt.split(",")[1:]:          # `int32_t a, b, c;`
                fields.append((extra.strip(), rust_type(first_type)))
        out.append("#[repr(C)]\n#[derive(Clone, Copy)]\npub struct " + rust_name(m.group(2)) + " {")
        out += [f"    pub {n}: {t}," for n, t in fields]
        out.append("}\n")
    out.append('extern "C" {')
    seen = set()
    for m in re.finditer(r"^\s*([A-Za-z_][A-Za-z0-9_ \*]*?)\s*\b(pi_[a-z0-9_]+)\s*\(([^;{]*?)\)\s*;", code, flags=re.M | re.S):
        ret, name, params = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        if name in seen:
            continue
        seen.add(name)
        args = []
        if params and params != "void":
            for p in params.split(","):
                t, n = split_decl(p)
                args.append(f"{n}: {rust_type(t)}")
        r = "" if ret == "void" else f" -> {rust_type(ret)}"
        out.append(f"    pub fn {name}({', '.join(args)}){r};")
    out.append("}")
    return "\n".join(out) + "\n"


if __name__ == "__main__":
    new = generate()
    if "--check" in sys.argv:
        sys.exit(0 if os.path.exists(OUT) and open(OUT).read() == new else 1)
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    open(OUT, "w").write(new)
    print(f"wrote {OUT}: {new.count('pub fn ')} functions")
