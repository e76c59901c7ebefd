"""The status word of linear attention, with a library that is made up: on the CPU."""

import contextlib

import pytest
import torch

from pararnn_b200 import _lib, ops


class Library:
    status = 0

    def prb_linear_attention_status(self, clear):
        s, Library.status = Library.status, 0 if clear else Library.status
        return s

    def prb_error_string(self, code):
        return b"made up"


@pytest.fixture
def library(monkeypatch):
    Library.status = 0
    monkeypatch.setattr(ops.L, "lib", lambda: Library())
    monkeypatch.setattr(ops, "_attention_devices", {torch.device("cuda", 0)})
    monkeypatch.setattr(ops, "_pending_backward", [])
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return Library


def test_a_backward_pass_behind_a_clean_check_is_looked_at(library):
    """Forward, check, backward (which registers nothing in Python), check."""
    ops.check_pending_backward()
    library.status = 1
    with pytest.raises(RuntimeError, match="bounded device-side wait.*linear attention"):
        ops.check_pending_backward()
    ops.check_pending_backward()


def test_an_error_of_the_device_is_not_taken_for_a_wait(library):
    library.status = -4
    with pytest.raises(RuntimeError, match="prb_linear_attention_status"):
        ops.check_pending_backward()


def test_nothing_is_asked_inside_a_capture(library, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    library.status = 1
    ops.check_pending_backward()
    assert library.status == 1


def test_the_words_are_empty_before_any_sweep():
    assert _lib.lib().prb_linear_attention_poll(1) == 0 and _lib.lib().prb_linear_attention_status(1) == 0
