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
    wrong, start = [0, 0], threading.Barrier(2)

    def work(i):
        stream = torch.cuda.Stream() if streams == 2 else torch.cuda.current_stream()
        start.wait(30)
        with torch.cuda.stream(stream):
            outs = [call(cases[i]) for _ in range(300)]
            stream.synchronize()
            wrong[i] = sum(not torch.equal(o, want[i]) for o in outs)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert wrong == [0, 0] and K.device_errors() == 0
