"""The C interface's version: one number in the header, the library and the package,
and the sizes of the params structs that go with it (a struct that changes needs a
new version, since an older caller's is shorter than what the library reads)."""
import os
import re

import pytest

from test_serving_cpu import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIZES = {101: dict(AtfPrefillParams=320, AtfDecodePlanParams=112, AtfDecodePlan=24, AtfDecodeParams=368, AtfMergeParams=104,
                   AtfRopeParams=152, AtfAppendParams=224, AtfExchangeParams=112, AtfPageTablesParams=160, AtfKvScales=32,
                   AtfPrefillRaggedPlanParams=32, AtfPrefillRaggedParams=216)}


def test_the_header_the_library_and_the_package_agree():
    ffi, lib = _lib()
    with open(os.path.join(ROOT, "include", "atflash_b200.h")) as f:
        version = int(re.search(r"^#define ATF_VERSION (\d+)$", f.read(), re.M).group(1))
    assert version == lib.atf_version() == ffi.ATF_VERSION
    assert {n: lib.atf_params_size(n.encode()) for n in SIZES[version]} == SIZES[version]


def test_a_library_of_another_version_is_refused(monkeypatch):
    ffi, _ = _lib()
    monkeypatch.setattr(ffi, "_lib", None)
    monkeypatch.setattr(ffi, "ATF_VERSION", ffi.ATF_VERSION + 1)
    with pytest.raises(ImportError, match="build it again"):
        ffi.load()
