"""Token-path operators without a GPU: refusals, registry, and the plain forms the GPU tests compare against."""

import numpy as np
import pytest
import torch

import difflut_b200 as difflut
from difflut_b200 import _native
from difflut_b200.encoder import EmbeddingEncoder, embedding_lookup
from difflut_b200.utils import Dropout, GroupNorm, dropout, group_norm, sample_logits
from difflut_b200.utils.warnings import DefaultValueWarning
from token_util import philox, sample_row


def test_philox_known_answers():
    """The published known-answer vectors of Philox4x32-10."""
    cases = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
             ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
             ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
              (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for counter, key, want in cases:
        got = philox(np.array([counter], dtype=np.uint64), key)[0]
        assert tuple(int(w) for w in got) == want


# ---------------------------------------------------------------------------------------------- embedding
def test_embedding_encoder_is_registered_and_has_nothing_to_fit():
    assert difflut.REGISTRY.get_encoder("embedding") is EmbeddingEncoder
    enc = EmbeddingEncoder(10, num_bits=4, scale=2.0, padding_idx=-1)
    assert enc.is_fitted and enc.fit(None) is enc
    assert list(enc.state_dict()) == ["weight"] and enc.weight.shape == (10, 4)
    assert float(enc.weight[-1].detach().abs().max()) == 0.0
    scaled = enc.weight.detach()[:-1] * 2.0
    assert float(scaled.min()) >= 0.0 and float(scaled.max()) < 1.0
    assert enc.to("cpu") is enc and isinstance(enc.weight, torch.nn.Parameter)
    assert "padding_idx=-1" in repr(enc)


@pytest.mark.parametrize("kwargs", [{"num_embeddings": 0}, {"num_embeddings": 2.5}, {"num_embeddings": 4, "scale": 0.0},
                                    {"num_embeddings": 4, "scale": float("nan")},
                                    {"num_embeddings": 4, "padding_idx": 4}, {"num_embeddings": 4, "padding_idx": -5}])
def test_embedding_encoder_refuses(kwargs):
    with pytest.raises(ValueError):
        EmbeddingEncoder(**kwargs)


def test_embedding_lookup_refuses():
    ids, weight = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        embedding_lookup(ids, weight)
    with pytest.raises(TypeError, match="int32 or int64"):
        embedding_lookup(ids.float(), weight)
    with pytest.raises(TypeError, match="int32 or int64"):
        embedding_lookup([1, 2], weight)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        embedding_lookup(ids, weight.double())
    with pytest.raises(ValueError, match="non-empty"):
        embedding_lookup(ids, weight[0])
    with pytest.raises(ValueError, match="non-empty"):
        embedding_lookup(ids, weight[:0])
    with pytest.raises(TypeError):
        EmbeddingEncoder(4, dtype=torch.float64)


def test_embedding_entry_points_refuse_bad_sizes():
    lib = _native.lib()
    for size in (lib.dl_embedding_bwd_scratch_bytes, lib.dl_embedding_order_bytes):
        assert size(100, 10, 8, 0) > 0 and size(0, 10, 8, 0) > 0
        for bad in ((-1, 10, 8, 0), (100, 0, 8, 0), (100, 10, 0, 0), (100, 10, 8, 3), (1 << 31, 10, 8, 0),
                    (100, 1 << 31, 8, 0)):
            assert size(*bad) == 0
    assert lib.dl_embedding(None, 64, None, None, 3, 4, 2, 0, 1.0, -1, None, None) == -1
    assert lib.dl_embedding(None, 64, None, None, 0, 4, 2, 0, 1.0, -1, None, None) == 0
    assert lib.dl_embedding(None, 16, None, None, 0, 4, 2, 0, 1.0, -1, None, None) == -1
    assert lib.dl_embedding(8, 64, 18, 16, 3, 4, 2, 0, 1.0, -1, None, None) == -4  # fp32 table at an odd half word
    assert lib.dl_embedding(8, 64, 16, 16, 3, 4, 2, 0, 1.0, -1, 64, None) == -4  # workspace not 256-byte aligned
    assert lib.dl_embedding(8, 64, 16, 16, 1 << 31, 4, 2, 0, 1.0, -1, 256, None) == -5
    assert lib.dl_embedding_bwd(256, 16, 16, 3, 4, 2, 0, 1.0, 64, None) == -4
    assert lib.dl_embedding_bwd(None, 16, 16, 3, 4, 2, 0, 1.0, 256, None) == -1
    assert lib.dl_embedding_bwd(256, 16, 16, 1 << 31, 4, 2, 0, 1.0, 256, None) == -5


# ---------------------------------------------------------------------------------------------- dropout
def test_dropout_refuses():
    x = torch.zeros(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dropout(x, 0.5)
    for p in (-0.1, 1.5, float("nan"), "0.5", True):
        with pytest.raises(ValueError, match="probability"):
            dropout(x, p)
    for name in ("seed", "offset"):
        for value in (-1, 1 << 63, 0.5, True):
            with pytest.raises(ValueError, match=name):
                dropout(x, 0.5, **{name: value})
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        dropout(x.double(), 0.5)


def test_dropout_module_host_side():
    import copy

    with pytest.warns(DefaultValueWarning):
        assert Dropout().p == 0.5
    with pytest.raises(ValueError):
        Dropout(2.0)
    d = Dropout(0.3)
    x = torch.ones(3)
    assert d.eval()(x) is x and Dropout(0.0).train()(x) is x
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        d.train()(x)
    assert copy.deepcopy(d).p == 0.3 and list(d.state_dict()) == []


def test_dropout_entry_points_refuse():
    lib = _native.lib()
    assert lib.dl_dropout(None, None, 0, 0, 0.5, 1, 0, None, None) == 0
    assert lib.dl_dropout(None, None, 4, 0, 0.5, 1, 0, None, None) == -1
    assert lib.dl_dropout(None, None, 0, 0, 1.5, 1, 0, None, None) == -1
    assert lib.dl_dropout(None, None, 0, 7, 0.5, 1, 0, None, None) == -1
    assert lib.dl_dropout(6, 8, 4, 0, 0.5, 1, 0, None, None) == -4
    assert lib.dl_counter_draw(None, None, None) == -1
    assert lib.dl_dropout(8, 8, 4, 0, 0.5, 1, 0, 12, None) == -4 and lib.dl_counter_draw(8, 12, None) == -4


# ---------------------------------------------------------------------------------------------- group norm
def test_group_norm_refuses():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm(x, 2)
    for groups in (0, 3, -2, 2.0, True):
        with pytest.raises(ValueError):
            group_norm(x, groups)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 2, activation="tanh")
    with pytest.raises(ValueError, match="eps"):
        group_norm(x, 2, eps=float("nan"))
    with pytest.raises(ValueError, match="weight"):
        group_norm(x, 2, w[:7])
    with pytest.raises(ValueError, match="bias"):
        group_norm(x, 2, w, w.view(1, 8))
    with pytest.raises(TypeError, match="weight"):
        group_norm(x, 2, w.half())
    with pytest.raises(TypeError, match="one type"):
        group_norm(x.half(), 2, w, w.half())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        group_norm(x.double(), 2)
    with pytest.raises(ValueError, match="shape"):
        group_norm(x[0, 0], 2)


def test_group_norm_module_host_side():
    for kwargs in ({"num_groups": 3}, {"num_groups": 0}, {"eps": -1.0}, {"activation": "gelu"}, {"channel_dim": 2}):
        with pytest.raises(ValueError):
            GroupNorm(**{"num_groups": 2, "num_channels": 8, **kwargs})
    m = GroupNorm(2, 8, activation="sigmoid", channel_dim=1)
    assert list(m.state_dict()) == ["weight", "bias"] and GroupNorm(2, 8, affine=False).weight is None
    with pytest.raises(ValueError, match="8 channels"):
        m(torch.zeros(2, 3, 8))
    assert "sigmoid" in repr(m)


def test_group_norm_entry_points_refuse():
    lib = _native.lib()
    for size in (lib.dl_group_norm_scratch_bytes, lib.dl_group_norm_bwd_scratch_bytes):
        assert size(2, 3, 8, 2, 0) >= 0 and size(0, 3, 8, 2, 0) >= 0 and size(2, 1, 100000, 1, 1) >= 0
        for bad in ((-1, 3, 8, 2, 0), (2, 0, 8, 2, 0), (2, 3, 0, 2, 0), (2, 3, 8, 3, 0), (2, 3, 8, 2, 5)):
            assert size(*bad) == -1
    assert lib.dl_group_norm_scratch_bytes(2, 1000, 64, 2, 0) > 0  # chunks of rows leave their sums there
    zeros = [None] * 7
    assert lib.dl_group_norm(*zeros, 2, 3, 8, 2, 0, 0, 0, 1e-5, None) == -1
    assert lib.dl_group_norm(*zeros, 0, 3, 8, 2, 0, 0, 0, 1e-5, None) == 0
    assert lib.dl_group_norm(*zeros, 0, 3, 8, 2, 0, 0, 4, 1e-5, None) == -1
    assert lib.dl_group_norm(16, None, None, 18, None, None, None, 2, 3, 8, 2, 0, 0, 0, 1e-5, None) == -4
    assert lib.dl_group_norm(16, None, None, 16, 16, None, None, 2, 3, 8, 2, 0, 0, 0, 1e-5, None) == -1
    assert lib.dl_group_norm(16, None, None, 16, None, None, None, 2, 1000, 64, 2, 0, 0, 0, 1e-5, None) == -1
    assert lib.dl_group_norm_bwd(*([16] * 10), 2, 3, 8, 2, 0, 0, 9, None) == -1
    assert lib.dl_group_norm_bwd(16, 16, None, None, None, 16, 16, 16, 16, 16, 2, 3, 8, 2, 0, 0, 0, None) == -1
    assert lib.dl_group_norm_bwd(*([16] * 9), None, 2, 3, 8, 2, 0, 0, 0, None) == -1
    for odd in (1, 2, 4, 5):  # weight, bias, mean, rstd
        args = [16, 16, 16, 16, 16, 16, 16]
        args[odd] = 18
        assert lib.dl_group_norm(*args, 2, 3, 8, 2, 0, 0, 0, 1e-5, None) == -4
    for odd in (2, 3, 4, 5, 7, 8):  # and the parameters' gradients
        args = [16] * 10
        args[odd] = 18
        assert lib.dl_group_norm_bwd(*args, 2, 3, 8, 2, 0, 0, 0, None) == -4


def test_group_norm_refuses_sizes_past_its_indexes():
    from difflut_b200.utils.normalization import _scratch_bytes

    for size in ((1, 1 << 30, 1, 1, 1), (1, 1, 1 << 30, 1, 1)):
        with pytest.raises(RuntimeError, match="not supported"):
            _scratch_bytes(*size)


# ---------------------------------------------------------------------------------------------- sampling
def test_sample_logits_refuses():
    x, u = torch.zeros(3, 5), torch.zeros(3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sample_logits(x, u)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        sample_logits(x.double(), u)
    with pytest.raises(ValueError, match="classes"):
        sample_logits(x[0], u)
    with pytest.raises(ValueError, match="classes"):
        sample_logits(x[:, :0], u)
    with pytest.raises(TypeError, match="u must"):
        sample_logits(x, u.half())
    with pytest.raises(TypeError, match="u must"):
        sample_logits(x, [0.0] * 3)
    with pytest.raises(ValueError, match="u must"):
        sample_logits(x, u[:2])
    with pytest.raises(ValueError, match="integers"):
        sample_logits(x, u, top_k=torch.ones(3))
    nan = float("nan")
    for name, values in (("temperature", (-1.0, nan, "1", True, torch.ones(2))), ("top_k", (-1, 1.5, True, torch.ones(3, 1))),
                         ("top_p", (0.0, 1.1, nan, -0.5)), ("min_p", (-0.1, 1.5, nan))):
        for value in values:
            with pytest.raises(ValueError, match=name):
                sample_logits(x, u, **{name: value})


def test_sample_entry_point_refuses():
    f = _native.lib().dl_sample_rows

    def call(logits=16, u=16, out=16, T=1.0, k=0, p=1.0, m=0.0, R=2, V=4, dtype=0):
        return f(logits, 4, u, 0, None, T, None, k, None, p, None, m, out, R, V, dtype, None)

    assert call(R=0) == 0 and call(logits=None) == -1 and call(u=None) == -1 and call(out=None) == -1
    assert call(V=0) == -1 and call(R=-1) == -1 and call(dtype=3) == -1 and call(V=1 << 30) == -5
    assert call(T=-1.0) == -1 and call(T=float("nan")) == -1 and call(k=-1) == -1
    assert call(p=0.0) == -1 and call(p=float("nan")) == -1 and call(m=-1.0) == -1 and call(m=1.5) == -1
    assert call(logits=18) == -4 and call(u=18) == -4 and call(out=20) == -4
    for odd in range(4):
        t, k, p, m = (18 if odd == i else None for i in range(4))
        assert f(16, 4, 16, 0, t, 1.0, k, 0, p, 1.0, m, 0.0, 16, 2, 4, 0, None) == -4


def test_plain_sampling_form_on_known_answers():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [sample_row(x, u) for u in (0.0, 0.0999, 0.1001, 0.4999, 0.5001, 0.6999, 0.7001)] == [0, 0, 1, 1, 2, 2, 3]
    assert sample_row(x, 0.99, k=1) == 1 and sample_row(x, 0.0, k=2) == 1 and sample_row(x, 0.9, k=2) == 3
    assert sample_row(x, 0.0, p=0.39) == 1 and sample_row(x, 0.9, p=0.41) == 3 and sample_row(x, 0.99, p=0.69) == 3
    assert sample_row(x, 0.0, min_p=0.6) == 1 and sample_row(x, 0.99, min_p=0.6) == 3
    assert sample_row(np.array([1.0, 2.0, 2.0]), 0.7, T=0) == 1
    assert sample_row(np.array([-np.inf, np.nan]), 0.5) == -1
    assert sample_row(np.array([0.0, np.inf, 1.0, np.inf]), 0.6) == 3
    assert sample_row(np.array([5.0, 5.0, 5.0]), 0.99, k=2) == 1 and sample_row(np.array([5.0, 5.0, 5.0]), 0.9, p=0.5) == 1
