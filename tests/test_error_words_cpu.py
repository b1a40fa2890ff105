"""CPU: every source with bounded waits has its error word wired to the host, read and cleared by the library."""
from __future__ import annotations

import glob
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "dynamic_conv1d_b200", "csrc")


def read(path):
    with open(path) as f:
        return f.read()


def test_every_error_word_is_reported():
    api = read(os.path.join(CSRC, "api.cu"))
    wiring, clearing, checking = (api[api.index(f):][:api[api.index(f):].index("\n}")]
                                  for f in ("void wire_host_error_word", "int report_earlier_timeout", "int dynconv_check_device"))
    words = {}
    for path in glob.glob(os.path.join(CSRC, "*.cu")):
        words.update(dict.fromkeys(re.findall(r"^DYNCONV_DEFINE_ERROR_ACCESSOR\((\w+)\)", read(path), re.M), path))
    assert len(words) >= 10
    for word, path in words.items():
        assert f"{word}_wire(mine)" in wiring and f"{word}()" in clearing and f"{word}()" in checking, path
    names = re.search(r"kFile\[\] = \{(.*?)\};", checking, re.S).group(1)
    assert len(re.findall(r'"[^"]+"', names)) == len(words)


def test_every_source_that_waits_has_one():
    """What calls a bounded wait, by itself or through a header that it includes, defines an accessor."""
    waits = re.compile(r"\bmbar_wait(_slow)?\(")
    headers = {os.path.basename(p): read(p) for p in glob.glob(os.path.join(CSRC, "*.cuh"))}
    waiting = {h for h, text in headers.items() if h != "common.cuh" and waits.search(text)}
    for path in glob.glob(os.path.join(CSRC, "*.cu")):
        text = read(path)
        if waits.search(text) or any(f'"{h}"' in text for h in waiting):
            assert "DYNCONV_DEFINE_ERROR_ACCESSOR" in text, path
