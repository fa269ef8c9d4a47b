#!/usr/bin/env python3
"""dev helper: build the library with extra -D switches.  usage: mkdef.py name [-DX=1 ...]  -> abx/lib<name>.so"""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from __graft_entry__ import compile_library  # noqa: E402

os.makedirs(os.path.join(ROOT, "abx"), exist_ok=True)
out = os.path.join(ROOT, "abx", f"lib{sys.argv[1]}.so")
compile_library(out, extra=sys.argv[2:])
print("built", out)
