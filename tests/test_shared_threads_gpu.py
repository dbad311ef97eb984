"""Attention over shared prefixes issued by two threads at once, on one stream and on two."""
import threading

import pytest
import torch

from shared_cases import PAGE, shared_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("streams", [1, 2])
@pytest.mark.parametrize("tc", [True, False])
def test_two_threads(tc, streams):
    from cima_b200.cache import LayerKV, SharedPrefixes
    from cima_b200.kernels import Kernels
    K = Kernels(verbose=False)
    cases = [shared_case([5], [4], [1, 64, 90], 28, 4, 64, torch.bfloat16, alone=[70], seed=s) for s in (1, 2)]

    def call(c):
        out = torch.empty(c.B, c.heads * c.hd, dtype=c.dtype, device="cuda")
        K.attention_shared(c.qkv, LayerKV(c.storage, c.table, PAGE, 0, 0, 0), c.slot, c.len, SharedPrefixes(c.order, c.own_page, c.groups, c.most), out, c.heads,
                           c.kv_heads, c.hd, c.scale, c.max_len, tc=tc)
        return out

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    wrong, start = [None, None], threading.Barrier(2)

    def work(i):
        try:
            stream = torch.cuda.Stream() if streams == 2 else torch.cuda.current_stream()
            start.wait(30)
            with torch.cuda.stream(stream):
                outs = [call(cases[i]) for _ in range(300)]
                stream.synchronize()
                wrong[i] = sum(not torch.equal(o, want[i]) for o in outs)
        except Exception as e:
            wrong[i] = e

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(isinstance(w, Exception) for w in wrong), wrong
    assert wrong == [0, 0] and K.device_errors() == 0


def test_a_thread_without_a_context():
    """A thread's first CUDA call may be a kernel that makes a tensor map."""
    from cima_b200.kernels import Kernels
    K = Kernels(verbose=False)
    a, w = torch.randn(256, 128, device="cuda").bfloat16(), torch.randn(256, 128, device="cuda").bfloat16()
    want, got = torch.empty(256, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(256, 256, dtype=torch.bfloat16, device="cuda")
    K.gemm_tc_pair(a, w, None, want, 0)
    K.device_errors()
    failed = []

    def work():
        try:
            K.gemm_tc_pair(a, w, None, got, 0)
        except Exception as e:
            failed.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join(60)
    assert not failed and torch.equal(got, want)
