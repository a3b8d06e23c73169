"""Embedding, attention on packed documents and norm clipping together, as a
training loop of a causal language model uses them (CPU; the same on the GPU
in gpu/test_packed_lm_gpu.py)."""
import os
import sys

import numpy as np

import anand_mxnet_amd as mx

sys.path.insert(0, os.path.dirname(__file__))
from packed_lm import check_documents, check_steps  # noqa: E402


def test_steps():
    check_steps(mx.cpu(), "float32")


def test_documents_are_apart():
    check_documents(mx.cpu(), "float32", 2e-5)
