"""CPU: argument checks of the operators on logits and of the sorted embedding gradient.  Nothing is launched: a call
with a bad argument is refused before the first CUDA call."""

import pytest

BAD, LIMIT = -1, -7
P = 4096                  # stands for an address: no call below gets as far as using it


@pytest.fixture(scope="module")
def L(built):
    from opennn_b200 import capi
    return capi.lib()


def logprobs(L, logits=P, dtype=0, pitch=100, tokens=P, logprobs=P, entropy=P, lse=P, ids=P, values=P, top=5, rows=4, V=100, T=1.0):
    return L.onn_token_logprobs(logits, dtype, pitch, tokens, logprobs, entropy, lse, ids, values, top, rows, V, T, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(dtype=3), dict(dtype=-1), dict(pitch=99), dict(rows=0), dict(rows=-1), dict(rows=1 << 27), dict(V=1), dict(V=0),
    dict(V=1 << 31, pitch=1 << 31), dict(ids=None), dict(values=None), dict(top=-1), dict(tokens=None),
    dict(logprobs=None, entropy=None, lse=None, top=0), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")),
    dict(logits=P + 2), dict(logits=P + 1, dtype=1)])
def test_token_logprobs_refuses(L, bad):
    assert logprobs(L, **bad) == BAD


def test_token_logprobs_limit(L):
    assert logprobs(L, top=129) == LIMIT


def backward(L, logits=P, dtype=0, pitch=100, tokens=P, lse=P, entropy=P, d_logprobs=P, d_entropy=P, out=P, d_pitch=100, rows=4, V=100, T=1.0):
    return L.onn_token_logprobs_bwd(logits, dtype, pitch, tokens, lse, entropy, d_logprobs, d_entropy, out, d_pitch, rows, V, T, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(tokens=None), dict(lse=None), dict(entropy=None), dict(d_logprobs=None), dict(out=None), dict(d_pitch=99),
    dict(out=P + 2), dict(out=P + 1, dtype=2), dict(T=0.0), dict(rows=0), dict(dtype=7), dict(d_pitch=101)])
def test_token_logprobs_bwd_refuses(L, bad):
    assert backward(L, **bad) == BAD


def distill(L, logits=P, dtype=0, pitch=100, targets=P, count=P, ids=P, values=P, top=5, T=2.0, soft=1.0, hard=0.5, out=P, d_pitch=100,
            stats=P, losses=P, rows=4, V=100):
    return L.onn_distill3d_fwd_bwd(logits, dtype, pitch, targets, count, ids, values, top, T, soft, hard, out, d_pitch, stats, losses, rows, V, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(targets=None), dict(ids=None), dict(values=None), dict(top=0), dict(stats=None), dict(losses=None),
    dict(T=0.0), dict(T=float("nan")), dict(soft=float("nan")), dict(hard=float("inf")), dict(d_pitch=99), dict(out=P + 2),
    dict(rows=0), dict(V=1), dict(d_pitch=101)])
def test_distill_refuses(L, bad):
    assert distill(L, **bad) == BAD


def test_distill_limit(L):
    assert distill(L, top=129) == LIMIT


def embed(L, ids=P, dY=P, dY2=P, dW=P, B=2, S=3, E=8, V=10, workspace=P, flags=0):
    return L.onn_embedding_bwd_sorted(ids, dY, dY2, dW, B, S, E, V, 1, workspace, flags, None)


@pytest.mark.parametrize("bad", [
    dict(ids=None), dict(dY=None), dict(dW=None), dict(B=0), dict(S=0), dict(E=0), dict(V=0), dict(V=1 << 24), dict(E=1 << 24),
    dict(B=1 << 20, S=1 << 12), dict(flags=8)])
def test_embedding_bwd_sorted_refuses(L, bad):
    assert embed(L, **bad) == BAD


def test_embedding_bwd_sorted_workspace(L):
    """Sizes do not need a GPU; a missing workspace is told from a bad argument."""
    assert L.onn_embedding_bwd_sorted_workspace_floats(2, 3, 8, 10) == 0
    floats = L.onn_embedding_bwd_sorted_workspace_floats(64, 256, 1024, 32000)
    assert floats >= 2 * 64 * 256
    assert L.onn_embedding_bwd_sorted_workspace_floats(0, 3, 8, 10) == 0
    assert embed(L, B=64, S=256, E=1024, V=32000, workspace=None) == -4
    assert embed(L, B=64, S=256, E=1024, V=32000, workspace=P + 4) == BAD


def test_wrappers_refuse_host_tensors(built):
    import torch

    from opennn_b200 import capi
    x, t = torch.zeros(2, 8), torch.ones(2)
    with pytest.raises(capi.OnnError):
        capi.token_logprobs(x, t)
    with pytest.raises(capi.OnnError):
        capi.token_logprobs(x.double(), t)
    with pytest.raises(capi.OnnError):
        capi.distill3d(x, t, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))


def test_tensors_of_another_device_are_refused(built):
    import torch

    from opennn_b200 import capi

    class On:
        """A tensor as the checks see it, on device `device`."""

        def __init__(self, device, dtype):
            self.device, self.dtype = device, dtype

        numel = staticmethod(lambda: 4)
        is_contiguous = staticmethod(lambda: True)
        data_ptr = staticmethod(lambda: 64)

        def get_device(self):
            return self.device

    assert capi._f32(On(1, torch.float32), 4, "tokens", 1) == 64 and capi._i32(On(0, torch.int32), 4, "ids", 0) == 64
    for call in (lambda: capi._f32(On(1, torch.float32), 4, "tokens", 0), lambda: capi._f32(On(-1, torch.float32), 4, "tokens", 0),
                 lambda: capi._i32(On(0, torch.int32), 4, "ids", 1), lambda: capi._f32(On(0, torch.float64), 4, "tokens", 0)):
        with pytest.raises(capi.OnnError):
            call()
