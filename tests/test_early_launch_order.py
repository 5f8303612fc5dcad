"""Kernels that begin while the one before them ends, by their sources: each waits for the earlier kernel before it lets a later one begin and
before it takes tensor memory. (Else a later kernel could begin, and read, before an earlier one than its own predecessor is done, and a kernel
could hold tensor memory that the kernel it waits for still asks for: both hang or read stale values only now and then, or with
another library's kernels, so that no run shows them.)"""
import re

import pytest

TAKES = ("tmem_alloc(", "tcgen05.alloc.")


def kernels(root):
    """(file, name, body without comments) of every kernel that waits or lets others begin."""
    for path in sorted((root / "fenix_b200" / "csrc").glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__ void\b", text):
            begin = text.index("{", text.index(") {", m.start()))
            depth, at = 0, begin
            while True:
                depth += {"{": 1, "}": -1}.get(text[at], 0)
                at += 1
                if depth == 0:
                    break
            body = text[begin:at]
            if "let_later_begin()" in body or "wait_for_earlier()" in body:
                yield path.name, re.sub(r"\s+", " ", text[m.end():begin])[:80], body


def test_early_kernels_wait_first(root):
    seen = []
    for file, name, body in kernels(root):
        seen.append(file)
        wait = body.find("wait_for_earlier();")
        assert wait >= 0, (file, name)
        assert body.count("{", 0, wait) - body.count("}", 0, wait) == 1, (file, name)  # every thread comes there
        let = body.find("let_later_begin();")
        assert let < 0 or let > wait, (file, name)
        for word in TAKES:
            take = body.find(word)
            assert take < 0 or wait < take, (file, name, word)
            assert take < 0 or let < 0 or take < let, (file, name, word)
    assert {"i8_pair.cu", "i8_rows.cu", "i8_stream.cu", "layer_norm.cu", "layer_norm_backward.cu"} <= set(seen)


@pytest.mark.parametrize("file", ["i8_stream.cu", "i8_pair.cu"])
def test_launches_that_may_begin_early(root, file):
    """A launch that allows it is of a kernel that waits."""
    text = (root / "fenix_b200" / "csrc" / file).read_text()
    assert "programmaticStreamSerializationAllowed = 1" in text and "wait_for_earlier();" in text


def test_tensor_memory_goes_before_the_cluster_waits(root):
    """A block of a cluster that held tensor memory while it waits for the others could keep it from one of them."""
    body = next(b for f, _, b in kernels(root) if f == "i8_stream.cu")
    assert 0 < body.find("tmem_dealloc(") < body.find("cluster_sync();")
