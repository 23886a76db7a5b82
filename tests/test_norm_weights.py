"""Where the norm weights of the prologues lie: their addresses go to the kernels
bare, so a weight on the host or on another GPU is refused before any call."""
import pytest
import torch

import fmkv


def test_weights_on_the_host_are_refused():
    w = torch.ones(128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        fmkv.make_prologue(w, 1e-6, 64, 1e4)
    for q, k in ((w, None), (None, w), (w, w)):
        with pytest.raises(ValueError, match="GPU"):
            fmkv.make_qkv_prologue(q, k, 1e-6, 64, 1e4)


class OtherGpu:
    """What the checks ask of a weight, on a GPU that is not the rows'."""

    device, shape = "cuda:7", (128,)

    def numel(self):
        return 128

    def get_device(self):
        return 7


@pytest.mark.gpu
def test_weights_on_another_gpu_are_refused(gpu):
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    q, k = (torch.ones((3, h, 128), dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    for weights in ((OtherGpu(), w), (w, OtherGpu())):
        pro = gpu.make_qkv_prologue(w, w, 1e-6, 64, 1e4)
        pro.weights = weights
        out = tuple(torch.full_like(x, 7.0) for x in (q, k)) + (None,)
        with pytest.raises(ValueError, match="cuda:7"):
            gpu.qkv_norm_rope(q, k, None, pos, pro, out=out)
        assert all(bool((o == 7.0).all()) for o in out[:2])
    pro = gpu.make_prologue(w, 1e-6, 64, 1e4)
    pro.weight = OtherGpu()
    cache = gpu.KVCache(gpu.make_desc(2, 128, 4, capacity=16))
    pool = gpu.PagedPool(gpu.make_desc(2, 128, 4), 2)
    table, zero = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    kk = k[:1]
    for call in (lambda: cache.append_projected(kk, kk, pro), lambda: cache.decode_step_projected(kk, kk, pro, q[0]),
                 lambda: pool.append_projected(kk[None], kk[None], table, zero, pro),
                 lambda: pool.decode_step_projected(kk[None], kk[None], table, zero, zero + 1, 1, pro, q[:1])):
        with pytest.raises(ValueError, match="cuda:7"):
            call()
    assert cache.offset() == 0
    torch.cuda.synchronize()
    assert not bool(pool.storage().any())
