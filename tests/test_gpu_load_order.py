"""A context that is created, loaded and sized while another part of the program keeps the default stream busy holds the
same weights as one that was loaded alone: nothing that prepares its buffers runs on a stream that its own does not
wait for."""
from __future__ import annotations

import os
import threading
from pathlib import Path

import numpy as np
import pytest

from minimind_orangepi_b200 import DecodeEngine
from minimind_orangepi_b200.synthetic import SHAPES, synthetic_prompt, write_runtime_model

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


class BusyDefaultStream:
    """Keeps a few milliseconds of work queued on the default stream: one thread that counts cycles, so that the GPU is
    free for others."""

    def __enter__(self):
        torch.cuda.synchronize()
        self.stop = threading.Event()
        self.running = threading.Event()
        self.thread = threading.Thread(target=self.work)
        self.thread.start()
        assert self.running.wait(60)
        return self

    def work(self):
        queue = []
        while not self.stop.is_set():
            torch.cuda._sleep(4_000_000)  # 2 ms
            e = torch.cuda.Event()
            e.record()
            queue.append(e)
            if len(queue) == 3:
                self.running.set()
                queue.pop(0).synchronize()

    def __exit__(self, *exc):
        self.stop.set()
        self.thread.join()
        torch.cuda.synchronize()


def answers(d, shape, n, cache=None):
    prompts = [synthetic_prompt(40 + i, 3 + 29 * i % 97, shape.vocab_size) for i in range(n)]
    with DecodeEngine(d, max_seqs=n, max_batch=n, packed_cache=cache) as e:
        seqs = [e.open_sequence(len(p) + 4) for p in prompts]
        first = e.prompt_pass(seqs, prompts)
        tokens, logits = e.step(seqs, [int(t) for t in first], want_logits=True)
        return first, tokens, logits, e.loaded_from


@pytest.mark.parametrize("persistent", ["0", "1"])
@pytest.mark.parametrize("n", [1, 5, 80])
def test_weights_loaded_beside_a_busy_default_stream(monkeypatch, tmp_path, n, persistent):
    monkeypatch.setenv("MMC_PERSISTENT", persistent)
    shape = SHAPES["minimind2-small"]
    d = write_runtime_model(Path("/tmp/mmc_test_models") / "load-order", shape, 17, eps=1e-5, theta=1e6)
    cache = tmp_path / "w.mmcpk"
    want = answers(d, shape, n)
    with BusyDefaultStream():
        got = answers(d, shape, n, cache)
        assert os.path.exists(cache)
        packed = answers(d, shape, n, cache)
    assert got[3] == "weights.bin" and packed[3] == "packed"
    for x in (got, packed):
        assert all(np.array_equal(a, b) for a, b in zip(x[:3], want[:3]))
