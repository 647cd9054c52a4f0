"""CPU: LeafPolicy is reached as the documents say, and its sizes."""
import importlib
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_name_of_the_documents_is_public():
    """README.md and INTEGRATION.md write pct_amd.<name>"""
    pct_amd = importlib.import_module("pct_amd")
    for doc in ("README.md", "INTEGRATION.md"):
        names = set(re.findall(r"\bpct_amd\.([A-Za-z_]+)\b", open(os.path.join(ROOT, doc)).read()))
        missing = sorted(n for n in names if not hasattr(pct_amd, n))
        assert names and not missing, (doc, missing)
    assert "LeafPolicy" in pct_amd.__all__
