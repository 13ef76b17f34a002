"""GPU tests of the prompt path from threads of a serving program: a thread whose first CUDA call is one
of these, several threads over one cache and one plan, each with its stream and workspace."""
import threading

import pytest
import torch

from test_gpu_prompt_path import Attend, Gather, Rotate

pytestmark = pytest.mark.gpu


def in_thread(*calls):
    """Each call in a fresh thread of its own, all at once; the first exception is raised here."""
    errors = []

    def guarded(f):
        try:
            f()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(f,)) for f in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


@pytest.mark.parametrize("kind", ["attend", "rotate", "gather"])
def test_first_call_of_a_thread(cuda_device, kind):
    r = {"attend": lambda: Attend([40, 9], [40, 300], 4, 2, 128, seed=1),
         "rotate": lambda: Rotate(40, 4, 2, 128, 128, seed=1),
         "gather": lambda: Gather([40, 9], [3, 0], 2, 128, seed=1)}[kind]()
    torch.cuda.synchronize()
    in_thread(r.run)
    r.check()


def test_threads_over_one_cache_and_plan(cuda_device):
    runs = [Attend([300 + i, 20], [300 + i, 900], 8, 2, 128, seed=i) for i in range(3)]
    turns = [Rotate(200 + i, 8, 2, 128, 128, seed=i, write=False) for i in range(3)]
    for r in runs:
        r.cache = runs[0].cache
    for r in turns:
        r.plan = turns[0].plan
    both = runs + turns
    outs = lambda r: r.out if isinstance(r, Attend) else r.q_out  # noqa: E731
    want = []
    for r in both:
        r.run()
        torch.cuda.synchronize()
        want.append(outs(r).clone())
        outs(r).fill_(7.0)
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()

    def loop(r, stream):
        def go():
            for _ in range(50):
                r.run(stream=stream.cuda_stream)
        return go
    in_thread(*(loop(r, s) for r, s in zip(both, streams)))
    torch.cuda.synchronize()
    for r, w in zip(both, want):
        assert torch.equal(outs(r), w)
        r.check()
