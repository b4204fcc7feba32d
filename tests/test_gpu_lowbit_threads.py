"""GPU: host threads that call the low-bit operators on one stream get what they get alone, bit for bit.

The calls of a layer or a cache share their scratch with those of other threads on the stream; each call's launches
have to stay together."""
import threading

import pytest
import torch

import megaqwen_b200 as mq

pytestmark = pytest.mark.gpu
CALLS = 300


def _rand(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").bfloat16()


def _together(*jobs):
    """Runs jobs (functions without arguments) CALLS times each in threads of their own, on the current stream; their results."""
    start, got, failed = threading.Barrier(len(jobs)), [[] for _ in jobs], []
    stream = torch.cuda.current_stream()

    def work(i):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(CALLS):
                    got[i].append(jobs[i]())
        except Exception as e:   # reported below; a thread's exception would be lost
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    return got


def _check(jobs):
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    for side in (False, True):
        with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
            for w, outs in zip(want, _together(*jobs)):
                assert len(outs) == CALLS and all(torch.equal(o, w) for o in outs)


def _layer(n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    return mq.Int8Linear(w, torch.rand(n, generator=g, device="cuda") * 1e-2)


def test_linear():
    """Two layers whose tokens differ in number, so that the scratch grows while they run, and one of few tokens."""
    a, b = _layer(256, 512, 1), _layer(300, 512, 2)
    xa, xb, xc = _rand((40, 512), 3), _rand((70, 512), 4), _rand((2, 512), 5)
    _check([lambda: a(xa), lambda: b(xb), lambda: a(xc)])


@pytest.mark.parametrize("tokens", [(20, 20), (20, 33), (1, 20), (1, 1)])
def test_attention_over_one_cache(tokens):
    """Chunks (two kernels and a workspace between them) and single tokens on the same cache."""
    B, S, H = 3, 900, 2
    c = mq.KV4Cache(1, B, S, num_kv_heads=H)
    c.append(0, _rand((B, S, H, 128), 1), _rand((B, S, H, 128), 2), torch.zeros(B, dtype=torch.int32, device="cuda"))
    n = torch.tensor([S, 500, 77], dtype=torch.int32, device="cuda")
    qa, qb = (_rand((B, t, 2 * H, 128), 5 + i) for i, t in enumerate(tokens))
    _check([lambda: c.attend(0, qa, n), lambda: c.attend(0, qb, n)])
    c.check_device()


def test_scratch_made_while_others_run():
    """Every call has another number of tokens, so the tables of sizes change under the threads."""
    B, S, H = 2, 300, 2
    c = mq.KV4Cache(1, B, S, num_kv_heads=H)
    c.append(0, _rand((B, S, H, 128), 1), _rand((B, S, H, 128), 2), torch.zeros(B, dtype=torch.int32, device="cuda"))
    n = torch.tensor([S, 171], dtype=torch.int32, device="cuda")
    q = _rand((B, 100, 2 * H, 128), 3)
    fresh = mq.KV4Cache(1, B, S, num_kv_heads=H)
    fresh.codes.copy_(c.codes)
    fresh.scales.copy_(c.scales)
    want = [c.attend(0, q[:, :t], n) for t in range(1, 101)]
    torch.cuda.synchronize()
    count = [0, 0]

    def job(i, step):
        t = count[i] * step % 100
        count[i] += 1
        return t, fresh.attend(0, q[:, :t + 1], n)

    for outs in _together(lambda: job(0, 1), lambda: job(1, 37)):
        assert all(torch.equal(o, want[t]) for t, o in outs)
