"""What the language model entry points take for overlapping memory."""

from __future__ import annotations

import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def overlap(fcv):
    return importlib.import_module(fcv.__name__ + ".lm")._overlap


def test_apart(overlap):
    buf = torch.zeros(10, 64)
    assert not overlap(buf[:5], buf[5:]) and not overlap(buf[5:], buf[:5])
    assert not overlap(buf[:, :32], buf[:, 32:]) and not overlap(buf[:, 32:], buf[:, :32])
    assert not overlap(buf[:, 8:16], buf[2:3, 16:64])            # a single row between the others
    heads = buf.view(10, 8, 8)
    assert not overlap(heads[:, :3], heads[:, 3:]) and not overlap(heads[:, 5:], buf[:, :40])
    assert not overlap(buf, torch.zeros(10, 64)) and not overlap(buf[:0], buf)
    assert not overlap(buf[0], buf[1])


def test_together(overlap):
    buf = torch.zeros(10, 64)
    assert overlap(buf, buf) and overlap(buf[:5], buf[4:]) and overlap(buf[4:], buf[:5])
    assert overlap(buf[:, :33], buf[:, 32:]) and overlap(buf[:, 32:], buf[:, :33])
    assert overlap(buf[:, 8:16], buf[2]) and overlap(buf[0, 3:], buf[0, :4])
    assert overlap(buf[1:, :32], buf.view(-1)[63:63 + 64 * 9].view(9, 64)[:, :32])
    assert overlap(buf[:, :8], buf.view(20, 32)[:, 8:16])        # at other strides: taken to
    assert overlap(buf[:1].expand(10, 64), buf[0])


def test_heads_between_heads(overlap):
    buf = torch.zeros(5, 6, 3, 8)                                # tokens, heads, q k v, dim
    q, k, v = buf[:, :, 0], buf[:, :, 1], buf[:, :, 2]
    assert not overlap(q, k) and not overlap(k, q) and not overlap(v, q) and not overlap(q[2:3], k)
    assert overlap(q, q[1:]) and overlap(q, q[:, 2:]) and overlap(v, v[3:4, 5:])
    assert overlap(q, buf[:, :, 0, 4:]) and overlap(buf[1:, :, 0], buf.flatten(1)[:4, 40:])
    last = buf.view(-1)[buf.stride(0) - 4:].as_strided((3, 8), (buf.stride(0), 1))  # past a row's end
    assert overlap(q[1:], last) and overlap(last, q[1:]) and not overlap(last, k[1:])
