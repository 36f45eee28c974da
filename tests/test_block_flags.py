"""The word that reports a product which gave up waiting, filled and read by
several threads (on the CPU: no kernel runs)."""
import threading
import time

import torch

from sdfoam_b200 import blocks


def unpinned(delay):
    """torch.zeros as the word's allocation asks for it, slow and not pinned."""
    zeros = torch.zeros

    def allocate(*args, pin_memory=False, **kw):
        time.sleep(delay)
        return zeros(*args, **kw)

    return allocate


def test_threads_that_meet_at_a_devices_first_product_share_its_word(monkeypatch):
    monkeypatch.setattr(blocks, "_flags", {})
    monkeypatch.setattr(torch, "zeros", unpinned(0.1))
    device, at, start = torch.device("cuda", 0), [None] * 4, threading.Barrier(4)

    def first(i):
        start.wait()
        at[i] = blocks._flag(device)

    threads = [threading.Thread(target=first, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert at == [blocks._flags[0][2]] * 4


def test_a_check_while_another_device_gets_its_word(monkeypatch):
    monkeypatch.setattr(blocks, "_flags", {})
    monkeypatch.setattr(torch, "zeros", unpinned(0.0))
    blocks._flag(torch.device("cuda", 0))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda index: blocks._flag(torch.device("cuda", index + 1))
                        if index < 3 else None)
    blocks.check_block_flags()
    assert 1 in blocks._flags
