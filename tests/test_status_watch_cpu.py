"""The watch over the status word, without a GPU: captures, results that take their time, another current device."""
import contextlib

import pytest
import torch

CODE = -4


class Fakes:
    def __init__(self):
        self.word = torch.zeros(1, dtype=torch.int32)
        self.capturing = set()                   # devices whose current stream is being captured
        self.current = 0
        self.copies = 0

    @contextlib.contextmanager
    def device(self, device):
        was, self.current = self.current, device.index
        yield
        self.current = was


@pytest.fixture
def fakes(monkeypatch):
    from tmq_b200 import ops
    f = Fakes()

    def word(device):
        f.copies += 1
        return f.word

    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    monkeypatch.setattr(ops, "gemm_status_word", word)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: f.current in f.capturing)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: f.current)
    monkeypatch.setattr(torch.cuda, "device", f.device)
    return f


@pytest.fixture
def watch(fakes):
    from tmq_b200 import ops
    return ops._StatusWatch(torch.device("cuda", 0))


def healthy(watch, n):
    for _ in range(n):
        watch.note_launch()


def test_the_first_call_behind_a_finished_copy_raises(fakes, watch):
    from tmq_b200 import _lib
    healthy(watch, 5)
    fakes.word.fill_(CODE)
    calls = 0
    with pytest.raises(_lib.TmqError):
        for _ in range(2 * watch.EVERY):
            calls += 1
            watch.note_launch()
    # the copy is made by the call that falls due, the very next one reports it
    assert calls == watch.EVERY - 5 + 2
    assert int(fakes.word) == 0 and not watch.pending
    healthy(watch, 3 * watch.EVERY)


def test_a_copy_that_has_not_landed_is_left_alone(fakes, watch):
    from tmq_b200 import _lib
    watch.note_launch()
    assert watch.pending
    watch.word.value = watch.UNREAD
    before = fakes.copies
    healthy(watch, 3 * watch.EVERY)
    assert watch.pending and fakes.copies == before
    watch.word.value = CODE
    with pytest.raises(_lib.TmqError):
        watch.note_launch()


def test_no_copy_becomes_part_of_a_graph(fakes, watch):
    """Whichever launches are captured: none of them copies, and what fell due is copied by the next that is not."""
    watch.note_launch()
    for start in range(watch.EVERY + 2):
        fakes.capturing = {0}
        before = fakes.copies
        healthy(watch, start + 1)
        assert fakes.copies == before
        fakes.capturing = set()
        for calls in range(2 * watch.EVERY):
            watch.note_launch()
            if fakes.copies > before:
                break
        assert fakes.copies == before + 1
        assert calls <= max(0, watch.EVERY - 1 - start)


def test_a_capture_neither_raises_nor_loses_a_failure(fakes, watch):
    from tmq_b200 import _lib
    watch.note_launch()
    assert watch.pending
    watch.word.value = CODE
    fakes.capturing = {0}
    healthy(watch, 2 * watch.EVERY)
    fakes.capturing = set()
    with pytest.raises(_lib.TmqError):
        watch.note_launch()


def test_every_eighth_launch_outside_captures_is_enough(fakes, watch):
    """A program that captures all but a few of its launches still hears of a failure."""
    from tmq_b200 import _lib
    healthy(watch, 2)
    fakes.word.fill_(CODE)
    outside = 0
    with pytest.raises(_lib.TmqError):
        for i in range(64 * watch.EVERY):
            fakes.capturing = set() if i % 8 == 3 else {0}
            outside += i % 8 == 3
            watch.note_launch()
    assert outside <= 2 * watch.EVERY


def test_the_launch_device_counts_not_the_current_one(fakes, watch):
    fakes.current = 1
    before = fakes.copies
    fakes.capturing = {0}                        # the watch's own device captures
    watch.note_launch()
    assert fakes.copies == before and fakes.current == 1
    fakes.capturing = set()
    watch.note_launch()
    assert fakes.copies == before + 1 and fakes.current == 1
