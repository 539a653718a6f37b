"""Scoring calls of several host threads on one handle."""
import pytest

pytestmark = pytest.mark.gpu


def test_calls_of_several_host_threads(sampler):
    """Taken ones and refused ones: results, counts and messages."""
    import threading

    import torch

    from minisample import MiniSampleError

    n, reps = 4, 200
    xs = [torch.randn(6, 1201, device="cuda") for _ in range(n)]
    tok = torch.randint(0, 1201, (6,), device="cuda", dtype=torch.int32)
    want = [sampler.logprobs(x, tok, top_n=4, entropy=True) for x in xs]
    torch.cuda.synchronize()
    before = sampler.launch_count()
    wrong = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(reps):
                got = sampler.logprobs(xs[i], tok, top_n=4, entropy=True)
                try:
                    sampler.logprobs(xs[i], tok, temperature=-1.0)
                    wrong.append("taken")
                except MiniSampleError as e:
                    if "temperature" not in str(e):
                        wrong.append(str(e))
            st.synchronize()
        if not all(torch.equal(a, b) for a, b in zip(got, want[i]) if a is not None):
            wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    assert sampler.launch_count() - before == n * reps
