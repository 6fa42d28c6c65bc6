#!/usr/bin/env python3
"""Generates rust/src/device/cuda_ffi.rs (the `extern "C"` block over libtlcuda) from
include/tlcuda.h, so that the Rust side cannot drift from the C header.

    python rust/gen_ffi.py            # rewrite the file
    python rust/gen_ffi.py --check    # exit 1 if the file on disk is stale
"""
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "tlcuda.h")
OUT = os.path.join(ROOT, "rust", "src", "device", "cuda_ffi.rs")

PRIM = {"int32_t": "i32", "int64_t": "i64", "uint32_t": "u32", "uint64_t": "u64", "size_t": "usize", "float": "f32",
        "double": "f64", "char": "c_char", "void": "c_void", "uint8_t": "u8", "int": "i32"}


def camel(name: str) -> str:
    special = {"qtensor": "QTensor", "kvcache": "KvCache", "kvcache8": "KvCache8"}
    return "Tlc" + "".join(special.get(p, p.capitalize()) for p in name[4:].split("_"))


def rust_type(t: str) -> str:
    """C type -> Rust.  Handles `const T *`, `T **` and `T *const *` (a pointer to const pointers)."""
    t = t.strip()
    pointee_const = t.startswith("const ")      # is what the NEXT pointer points to const?
    if pointee_const:
        t = t[6:].strip()
    m = re.match(r"([\w ]+?)\s*((?:\*\s*(?:const\s*)?)*)$", t)
    base, ptrs = m.group(1).replace("struct ", "").strip(), m.group(2)
    r = PRIM.get(base) or (camel(base) if base.startswith("tlc_") else base)
    levels = re.findall(r"\*\s*(const)?", ptrs)
    if not levels:
        return "()" if r == "c_void" else r
    out = r
    for qual in levels:
        out = ("*const " if pointee_const else "*mut ") + out
        pointee_const = qual == "const"
    return out


def prototypes(header: str):
    h = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    for p in re.findall(r"TLC_API\s+(.*?);", h, flags=re.S):
        if p.lstrip().startswith("#") or "define" in p:
            continue
        p = " ".join(p.split())
        m = re.match(r"(.*?)\b(tlc_\w+)\s*\((.*)\)$", p)
        ret, name, args = m.group(1), m.group(2), m.group(3)
        params = []
        if args.strip() != "void":
            for a in args.split(","):
                mm = re.match(r"(.*?)(\w+)$", a.strip())
                ty, an = mm.group(1), mm.group(2)
                params.append(("ty" if an == "type" else an, rust_type(ty)))
        yield name, params, rust_type(ret)


def opaque_types(header: str):
    return sorted(set(re.findall(r"typedef struct (tlc_\w+) \1;", header)))


def structs(header: str):
    """Plain-data structs of the header (typedef struct name { ... } name;) as #[repr(C)]."""
    out = []
    for name, body in re.findall(r"typedef struct (tlc_\w+)\s*\{(.*?)\}\s*\1;", header, flags=re.S):
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            ty, names = decl.rsplit(" ", 1)[0], decl
            m = re.match(r"(\w+(?: \w+)*?) ((?:\w+(?:, )?)+)$", decl)
            ty, names = m.group(1), m.group(2)
            for n in names.split(","):
                fields.append((n.strip(), rust_type(ty)))
        out.append((name, fields))
    return out


def render() -> str:
    header = open(HEADER).read()
    lines = ["// GENERATED by rust/gen_ffi.py from include/tlcuda.h -- do not edit.",
             "//",
             "// The C ABI of libtlcuda: what takes the place of the MetalDevice / MetalBuffer /",
             "// KernelExecutor calls of src/device/ in the TensorLogic crate.  Every function returns",
             "// a status (0 = ok, negative = the TensorError variant named in TlcStatus below);",
             "// tlc_last_error() gives the message of the last failure on the calling thread.",
             "#![allow(non_camel_case_types, dead_code)]",
             "use std::os::raw::{c_char, c_void};", ""]
    for t in opaque_types(header):
        lines += ["#[repr(C)]", f"pub struct {camel(t)} {{ _private: [u8; 0] }}"]
    lines.append("")
    for name, fields in structs(header):
        lines += ["#[repr(C)]", "#[derive(Clone, Copy, Debug, Default)]", f"pub struct {camel(name)} {{"]
        lines += [f"    pub {n}: {t}," for n, t in fields]
        lines += ["}", ""]
    for m in re.finditer(r"^\s*(TLC_(?:OK|ERR_\w+|TYPE_\w+|SPLIT_\w+))\s*=\s*(-?\d+)", header, flags=re.M):
        lines.append(f"pub const {m.group(1)}: i32 = {m.group(2)};")
    lines += ["", '#[link(name = "tlcuda")]', 'extern "C" {']
    for name, params, ret in prototypes(header):
        sig = f"    pub fn {name}(" + ", ".join(f"{n}: {t}" for n, t in params) + ")" + ("" if ret == "()" else f" -> {ret}") + ";"
        if len(sig) > 110:
            head = f"    pub fn {name}("
            cur, out = head, []
            for i, (n, t) in enumerate(params):
                piece = f"{n}: {t}" + (", " if i < len(params) - 1 else "")
                if len(cur) + len(piece) > 108:
                    out.append(cur.rstrip())
                    cur = " " * len(head) + piece
                else:
                    cur += piece
            out.append(cur + ")" + ("" if ret == "()" else f" -> {ret}") + ";")
            sig = "\n".join(out)
        lines.append(sig)
    lines += ["}", ""]
    return "\n".join(lines)


def main() -> int:
    text = render()
    if "--check" in sys.argv:
        ok = os.path.exists(OUT) and open(OUT).read() == text
        print("cuda_ffi.rs is up to date" if ok else "cuda_ffi.rs is STALE: run python rust/gen_ffi.py")
        return 0 if ok else 1
    with open(OUT, "w") as f:
        f.write(text)
    print(OUT)
    return 0


if __name__ == "__main__":
    sys.exit(main())
