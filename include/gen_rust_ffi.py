#!/usr/bin/env python3
"""Rust `extern "C"` declarations for every function include/ttt_b200.h declares.

    python include/gen_rust_ffi.py            # prints the block
    python include/gen_rust_ffi.py --update   # rewrites the block between the markers in the integration guide

The block in the integration guide is generated, never edited by hand; tests/test_abi_host.py regenerates it and compares, and
checks every declaration's argument count against the ctypes table the Python binding uses.
"""

from __future__ import annotations

import re
import sys
from pathlib import Path
from typing import List, Tuple

HERE = Path(__file__).resolve().parent
HEADER = HERE / "ttt_b200.h"
DOC = HERE.parent / "INTEGRATION.md"
BEGIN = "<!-- generated by include/gen_rust_ffi.py: begin -->"
END = "<!-- generated by include/gen_rust_ffi.py: end -->"

_TYPES = {
    "const ttt_dims*": "*const TttDims", "const ttt_rotation*": "*const TttRotation", "const void*": "*const c_void", "void*": "*mut c_void",
    "const float*": "*const f32", "const int64_t*": "*const i64", "float*": "*mut f32", "const char*": "*const c_char",
    "size_t": "usize", "int64_t": "i64", "int32_t": "i32", "uint32_t": "u32", "int": "c_int", "float": "f32",
}


def declarations(text: str = None) -> List[Tuple[str, str, List[Tuple[str, str]]]]:
    """[(return type, name, [(type, name), ...])] of the header's function declarations, in header order."""
    text = HEADER.read_text() if text is None else text
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    text = re.sub(r"//[^\n]*", " ", text)
    text = re.sub(r"^\s*#.*$", " ", text, flags=re.M)
    body = text[text.index('extern "C" {') + len('extern "C" {'):]
    out = []
    for m in re.finditer(r"([A-Za-z_][\w\s\*]*?)\b(ttt_\w+)\s*\(([^;{}]*)\)\s*;", body):
        ret, name, args = " ".join(m.group(1).split()), m.group(2), " ".join(m.group(3).split())
        params = []
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                mm = re.match(r"(.*?)(\w+)$", a)
                ty = mm.group(1).replace(" *", "*").strip()
                params.append((ty, mm.group(2)))
        out.append((ret.replace(" *", "*"), name, params))
    return out


def rust_block() -> str:
    lines = ['#[link(name = "ttt_b200")]', 'extern "C" {']
    for ret, name, params in declarations():
        args = ", ".join(f"{n}: {_TYPES[t]}" for t, n in params)
        r = "" if ret == "void" else f" -> {_TYPES[ret]}"
        decl = f"    pub fn {name}({args}){r};"
        if len(decl) <= 118:
            lines.append(decl)
        else:  # wrap the argument list
            cur, rows = "        ", []
            for piece in [p + "," for p in args.split(", ")]:
                if len(cur) + len(piece) + 1 > 118:
                    rows.append(cur.rstrip())
                    cur = "        "
                cur += piece + " "
            rows.append(cur.rstrip().rstrip(","))
            lines.append(f"    pub fn {name}(")
            lines.extend(rows)
            lines.append(f"    ){r};")
    lines.append("}")
    return "\n".join(lines)


def doc_block() -> str:
    return f"{BEGIN}\n```rust\n{rust_block()}\n```\n{END}"


def current_doc_block() -> str:
    s = DOC.read_text()
    return s[s.index(BEGIN):s.index(END) + len(END)]


if __name__ == "__main__":
    if "--update" in sys.argv:
        s = DOC.read_text()
        a, b = s.index(BEGIN), s.index(END) + len(END)
        DOC.write_text(s[:a] + doc_block() + s[b:])
        print(f"updated {DOC}")
    else:
        print(rust_block())
