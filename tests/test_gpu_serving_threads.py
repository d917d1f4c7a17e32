"""Calls of different threads on different caches do not disturb one another."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _run(jobs):
    """Every job in a thread of its own, on a stream of its own; the first exception is raised here."""
    failed = []

    def guard(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                job()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=guard, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


def test_selections_of_different_length(cuda_device):
    """Numbers of blocks from 9,000 to 45,000, whose keys take different amounts of shared memory."""
    import smallaios_b200 as sa

    def job(blocks):
        past = blocks * 64 - 1
        cache = sa.GpuKvCache(1, 1, 16, past + 1, batch=1, num_heads=1, bits=4, device=cuda_device)
        cache.set_position(past)
        means = torch.zeros(1, 1, blocks, 16, dtype=torch.bfloat16, device=cuda_device)
        q = torch.ones(1, 1, 16, device=cuda_device)

        def run():
            for _ in range(400):
                ids = sa.gqa_select_blocks(q, cache, 0, means, num_heads=1, max_blocks=4)
            assert ids.tolist() == [[[[0, 1, 2, blocks - 1]]]]
        return run

    jobs = [job(n) for n in (9000, 16000, 30000, 45000)]
    torch.cuda.synchronize()
    for _ in range(3):
        _run(jobs)


def test_keeping_the_widest_drafts(cuda_device):
    """64 drafts of the widest format with QJL residuals, starting inside a 16-token block: the most shared memory."""
    import smallaios_b200 as sa

    past, n = 15, 64
    cache = sa.GpuKvCache(1, 1, 256, past + n, batch=1, num_heads=1, bits=8, qjl_residual=True, device=cuda_device)
    view = cache.view(0)
    for a in (view.k_codes, view.v_codes, view.k_qjl_bits, view.v_qjl_bits):
        a.random_(0, 256)
    for a in (view.k_meta, view.v_meta, view.k_qjl_mag, view.v_qjl_mag):
        a.normal_()
    cache.set_position(past)
    names = ("k_codes", "k_meta", "v_meta", "k_qjl_bits", "v_qjl_bits", "k_qjl_mag", "v_qjl_mag")
    before = {x: getattr(view, x).clone() for x in names} | {"v": view.v_codes_tokens().clone()}
    path = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=cuda_device)[None]
    cache.keep_drafts(path, drafted=n)
    for x, was in before.items():
        now = view.v_codes_tokens() if x == "v" else getattr(view, x)
        assert torch.equal(now[:, :, past:past + n], was[:, :, past:past + n].flip(2)), x
        assert torch.equal(now[:, :, :past], was[:, :, :past]), x
    cache.close()
