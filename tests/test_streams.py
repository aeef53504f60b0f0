"""Streams are created at the default priority: work on streams of different
priorities has hung MI355X machines for good."""
import ast
import inspect
import pathlib
import re

import pytest

import spmm_amd
from spmm_amd.parallel.loopback import PanelComm

ROOT = pathlib.Path(__file__).resolve().parent.parent
PACKAGE = pathlib.Path(spmm_amd.__path__[0])
PYTHON = [p for d in (PACKAGE, ROOT / "tools", ROOT / "benches", ROOT / "perf") for p in sorted(d.rglob("*.py"))]
PYTHON += sorted(ROOT.glob("*.py"))
NATIVE = [p for d in (PACKAGE / "csrc", ROOT / "tools") for p in sorted(d.rglob("*"))
          if p.suffix in (".hip", ".cpp", ".hpp", ".h")]
SCRIPTS = sorted((ROOT / "tools").rglob("*.sh"))


def priorities(path):
    """Keyword arguments of calls that give a stream or a process group a priority."""
    tree = ast.parse(path.read_text())
    return [f"{path.relative_to(ROOT)}:{n.lineno}" for n in ast.walk(tree) if isinstance(n, ast.Call)
            for k in n.keywords if k.arg and ("priority" in k.arg)]


def test_no_stream_gets_a_priority():
    assert len(PYTHON) > 30 and len(NATIVE) > 10
    assert [at for p in PYTHON for at in priorities(p)] == []
    assert [str(p) for p in NATIVE if re.search(r"StreamCreateWithPriority", p.read_text())] == []
    assert [str(p) for p in SCRIPTS if re.search(r"(?i)link-priority|SIDE_PRIO", p.read_text())] == []


def test_emulated_links_take_no_priority():
    assert "link_priority" not in inspect.signature(PanelComm.__init__).parameters
    with pytest.raises(TypeError, match="link_priority"):
        PanelComm(0, 1, None, [None], link_priority=-1)
