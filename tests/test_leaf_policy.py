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


def test_an_empty_batch_reaches_the_operators(monkeypatch):
    """no observations give no logits (heads are split by their width: a size to be inferred is refused for empty tensors)"""
    ops = importlib.import_module("online-3d-bpp-pct_amd.policy_ops")
    monkeypatch.setattr(ops, "_on_gpu", lambda name, *tensors: tensors[0].device)
    monkeypatch.setattr(ops, "_call", lambda *a: pytest.fail("nothing is launched for an empty batch"))
    net = importlib.import_module("pct_amd").LeafPolicy(8, 5, width=32, heads=2)
    logits = net(torch.zeros(0, 14, 9))
    assert logits.shape == (0, 5)
    logits.sum().backward()
    assert all(p.grad is not None and not p.grad.any() for p in net.parameters())
