"""The structs that INTEGRATION.md tells a Rust caller to declare are those of the headers, field by field."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _read(*path):
    return open(os.path.join(ROOT, *path), encoding="utf-8").read()


@pytest.mark.parametrize("rust,c", [("NvcRunnerOptions", "nvc_runner_options"), ("NvcQwen3Config", "nvc_qwen3_config")])
def test_structs(rust, c):
    kinds = {"i32": "int32_t", "f32": "float", "i64": "int64_t"}
    mine = [(n, kinds[t], int(size or 1)) for n, array, t, size in re.findall(r"pub (\w+): (\[)?(\w+)(?:; (\d+)\])?", re.search(r"pub struct %s \{(.*?)\n?\s*\}" % rust, _read("INTEGRATION.md"), re.S).group(1))]
    head = re.sub(r"/\*.*?\*/", "", _read("include", "nvc_b200_engine.h"), flags=re.S)
    theirs = []
    for kind, names in re.findall(r"(\w+)\s+([^;]+);", re.search(r"typedef struct %s \{(.*?)\}" % c, head, re.S).group(1)):
        for name, size in re.findall(r"(\w+)(?:\[(\d+)\])?", names):
            theirs.append((name, kind, int(size or 1)))
    assert mine == theirs
