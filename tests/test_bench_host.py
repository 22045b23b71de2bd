"""What the benchmark's line says of its measured traffic (CPU only)."""

from __future__ import annotations

import pathlib
import shutil
import sys

ROOT = pathlib.Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

import bench  # noqa: E402


def test_other_operators_do_not_make_the_traffic_stale(tmp_path, monkeypatch):
    """The traffic was measured on these attention sources.  Entry points of other
    operators that the C ABI's file takes in change none of its kernels; a change of
    its own, or of a kernel, counts."""
    csrc = tmp_path / 'nitrix_amd' / 'csrc'
    shutil.copytree(ROOT / 'nitrix_amd' / 'csrc', csrc)
    monkeypatch.setattr(bench, '_ROOT', str(tmp_path))
    now = bench._src_fingerprint(bench.ATTN_SOURCES)
    capi = csrc / 'nxa_capi.hip'
    text = capi.read_text()
    capi.write_text(text + '#include "nxa_capi_more.h"\n')
    assert bench._src_fingerprint(bench.ATTN_SOURCES) == now
    capi.write_text(text + 'int more;\n')
    assert bench._src_fingerprint(bench.ATTN_SOURCES) != now
    capi.write_text(text)
    kernel = csrc / 'nxa_fwd16.hip'
    kernel.write_text(kernel.read_text() + '\n')
    assert bench._src_fingerprint(bench.ATTN_SOURCES) != now
