"""CPU tests of the ranking-head operators: refusals, the modules' parameters, and the C entry points'
checks of their arguments (none of which touches a GPU)."""
import ctypes

import pytest
import torch

from collie_amd import _lib, functional as F, layers, ops


def test_modules_have_the_parameters_of_their_torch_counterparts():
    assert dict(layers.LayerNorm(8).named_parameters()).keys() == {'weight', 'bias'}
    assert layers.LayerNorm(8, elementwise_affine=False).weight is None
    lin = layers.Linear(8, 3, activation='gelu')
    lin.load_state_dict(torch.nn.Linear(8, 3).state_dict())
    names = [n for n, _ in layers.GatedLinear(8, 3).named_parameters()]
    assert names == ['gate.weight', 'gate.bias', 'up.weight', 'up.bias']
    assert len(list(layers.GatedLinear(8, 3, bias=False).parameters())) == 2
    for cls in (layers.Linear, layers.GatedLinear):
        with pytest.raises(ValueError, match='is not an activation'):
            cls(8, 3, activation='tanh')
    with pytest.raises(ValueError, match='last dimension only'):
        layers.LayerNorm((4, 8))
    with pytest.raises(ValueError, match='expected'):
        layers.LayerNorm(8)(torch.zeros(2, 7))


def test_no_cpu_fallback():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    for call in (lambda: F.layer_norm(x), lambda: F.linear(x, w), lambda: F.gated_linear(x, w, w),
                 lambda: F.embedding_rows(w, torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.embedding_rows_grad(torch.zeros(2, dtype=torch.int64), x, 3)):
        with pytest.raises(_lib.CollieHipError, match='no CPU fallback'):
            call()


def test_tables_on_the_cpu_are_torch_embeddings():
    t = layers.ScaledEmbedding(5, 3)
    ids = torch.tensor([0, 4, 4])
    assert torch.equal(t(ids), torch.nn.functional.embedding(ids, t.weight))
    t(ids).sum().backward()
    assert t.weight.grad[4].tolist() == [2.0] * 3


def test_refusals_before_any_launch():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    with pytest.raises(ValueError, match='is not an activation'):
        F.linear(x, w, activation='softplus')
    with pytest.raises(ValueError, match='both or none'):
        F.gated_linear(x, w, w, torch.zeros(3), None)
    with pytest.raises(ValueError, match='eps'):
        F.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match='padding_idx'):
        F.embedding_rows(w, torch.zeros(1, dtype=torch.int64), padding_idx=3)
    with pytest.raises(_lib.CollieHipError, match='status'):
        F.embedding_rows(w, torch.zeros(1, dtype=torch.int64), status=torch.zeros(1))
    for call in (lambda: F.linear(x, w, torch.zeros(1, 3)), lambda: F.layer_norm(x, torch.zeros(3)),
                 lambda: F.gated_linear(x, w, torch.zeros(4, 3))):
        with pytest.raises(ValueError, match='must have shape'):
            call()
    with pytest.raises(ValueError, match='do not fit'):
        F.linear(x, torch.zeros(3, 5))
    with pytest.raises(ValueError, match='is empty'):
        F.linear(x, torch.zeros(0, 4))
    with pytest.raises(_lib.CollieHipError, match='bias is torch.float64, x is torch.float32'):
        F.linear(x, w, torch.zeros(3, dtype=torch.float64))
    with pytest.raises(_lib.CollieHipError, match='weight is torch.float32, bias is torch.bfloat16'):
        F.layer_norm(x.bfloat16(), torch.ones(4), torch.zeros(4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match='residual must have shape'):
        F.linear(x, w, residual=torch.zeros(1, 3))
    with pytest.raises(_lib.CollieHipError, match='residual is'):
        F.linear(x, w, residual=torch.zeros(2, 3, dtype=torch.bfloat16))
    with pytest.raises(_lib.CollieHipError, match='float64'):
        F.layer_norm(x.double())
    with pytest.raises(_lib.CollieHipError, match='index tensors'):
        F.embedding_rows(w, torch.zeros(2, dtype=torch.int16))
    for call in (lambda v: F.embedding_rows(v, torch.zeros(2, dtype=torch.int64)),
                 lambda v: F.layer_norm(v), lambda v: F.linear(v, v), lambda v: F.linear(x[:, :1], v.t()),
                 lambda v: ops.embedding_rows_grad(torch.zeros(1, dtype=torch.int64), v, 3)):
        with pytest.raises(ValueError, match='too wide'):
            call(torch.zeros(1, 1).expand(1, (1 << 32) + 8))
    with pytest.raises(ValueError, match='does not belong'):
        ops.embedding_rows_grad(torch.zeros(3, dtype=torch.int64), x, 5)


def test_rows_view_copies_only_what_it_must():
    rows_view = _lib.load_autograd().rows_view
    base = torch.arange(60.0).reshape(5, 12)
    t, ld = rows_view(base[:, 2:9], 7)
    assert t.data_ptr() == base[:, 2:].data_ptr() and ld == 12
    for view in (base.t(), base[:1, :7].expand(5, 7), base[:, ::2],
                 base.reshape(5, 3, 4)[:, 1:, :], base.as_strided((4, 8), (3, 1))):
        t, ld = rows_view(view, view.shape[-1])
        assert t.is_contiguous() and ld == t.shape[1]
        assert torch.equal(t.reshape(view.shape), view)
    assert rows_view(torch.zeros(7), 7)[0].shape == (1, 7)
    assert rows_view(torch.zeros(0, 3, 7), 7)[0].shape == (0, 7)


def test_c_entry_points_reject_bad_arguments():
    lib = _lib.load()
    p = ctypes.c_void_p(256)            # never dereferenced: every call below is refused
    none, big = ctypes.c_void_p(None), 1 << 40
    bad = [
        lambda: lib.collie_embedding_rows(p, 9, 4, 4, p, 1, 1, 1.0, p, none, none),
        lambda: lib.collie_embedding_rows(p, 0, 0, 4, p, 1, 1, 1.0, p, none, none),
        lambda: lib.collie_embedding_rows(p, 0, 4, 0, p, 1, 1, 1.0, p, none, none),
        lambda: lib.collie_embedding_rows(p, 0, 4, 4, p, 7, 1, 1.0, p, none, none),
        lambda: lib.collie_embedding_rows(none, 0, 4, 4, p, 1, 1, 1.0, p, none, none),
        lambda: lib.collie_embedding_rows(p, 0, 4, 4, p, 1, -1, 1.0, p, none, none),
        lambda: lib.collie_embedding_rows_grad(p, 1, 5, p, 3, 0, 4, 4, 1.0, -1, p, p, 1 << 30, none,
                                               none),
        lambda: lib.collie_embedding_rows_grad(p, 1, 5, p, 4, 0, 4, 4, 1.0, -1, p, p, 16, none, none),
        lambda: lib.collie_embedding_rows_grad(p, 1, 1 << 30, p, 4, 0, 4, 4, 1.0, -1, p, p, 1 << 60,
                                               none, none),
        lambda: lib.collie_embedding_rows_grad(p, 1, 5, p, 4, 0, 4, 4, 1.0, -1, ctypes.c_void_p(8),
                                               p, 1 << 30, none, none),
        lambda: lib.collie_layer_norm_forward(p, 3, 0, 2, 4, p, p, 0, 1e-5, p, p, p, none),
        lambda: lib.collie_layer_norm_forward(p, 4, 1, 2, 4, p, p, 2, 1e-5, p, p, p, none),
        lambda: lib.collie_layer_norm_forward(p, 4, 0, 2, 4, p, p, 0, -1.0, p, p, p, none),
        lambda: lib.collie_layer_norm_forward(p, 4, 0, 2, 4, p, p, 0, 1e-5, p, p, none, none),
        lambda: lib.collie_layer_norm_backward(p, 4, p, 4, 0, 2, 4, p, 0, none, p, p, p, p, p,
                                               1 << 30, none),
        lambda: lib.collie_layer_norm_backward(p, 4, p, 4, 0, 2, 4, p, 0, p, p, p, p, p, p, 4, none),
        lambda: lib.collie_linear_forward(p, 3, 0, 2, 4, p, p, 5, 0, none, 0, none, p, p, big, none),
        lambda: lib.collie_linear_forward(p, 4, 0, 2, 4, p, p, 5, 6, none, 0, none, p, p, big, none),
        lambda: lib.collie_linear_forward(p, 4, 0, 2, 4, p, p, 5, 0, p, 4, none, p, p, big, none),
        lambda: lib.collie_linear_forward(p, 4, 5, 2, 4, p, p, 5, 0, none, 0, none, p, p, big, none),
        lambda: lib.collie_linear_forward(p, 4, 0, 2, 4, p, p, 5, 0, none, 0, none, p, p, 1, none),
        lambda: lib.collie_gated_forward(p, 4, 0, 2, 4, p, p, p, p, 5, 4, p, p, p, none, big, none),
        lambda: lib.collie_gated_forward(p, 4, 0, 2, 4, p, p, p, none, 5, 4, none, none, p, p, big, none),
        lambda: lib.collie_gated_forward(p, 4, 0, 2, 4, p, p, none, none, 5, 4, p, none, p, p, big, none),
        lambda: lib.collie_linear_backward(p, 5, p, 4, 0, 0, 4, p, 5, 0, none, p, p, p, p, 1 << 30,
                                           none),
        lambda: lib.collie_linear_backward(p, 5, p, 4, 0, 2, 4, p, 5, 4, none, p, p, p, p, 1 << 30,
                                           none),
        lambda: lib.collie_linear_backward(p, 5, p, 4, 0, 2, 4, p, 5, 0, none, p, p, p, p, 1, none),
        lambda: lib.collie_gated_backward(p, 5, p, 4, 0, 2, 4, p, p, 5, 4, p, none, p, p, p, p, p, p,
                                          1 << 30, none),
        lambda: lib.collie_gated_backward(p, 4, p, 4, 0, 2, 4, p, p, 5, 4, p, p, p, p, p, p, p, p,
                                          1 << 30, none),
    ]
    for i, call in enumerate(bad):
        assert call() == -1, i
        assert lib.collie_last_error()


def _hybrid(**kw):
    from collie_amd.hybrid import HybridPretrainedModel
    from collie_amd.model import MatrixFactorizationModel

    class Shape:
        num_users, num_items, num_negative_samples = 30, 20, 3

    torch.manual_seed(1)
    mf = MatrixFactorizationModel(train=Shape(), embedding_dim=8, lr_scheduler_func=None)
    return HybridPretrainedModel(train=Shape(), item_metadata=torch.ones(20, 6), trained_model=mf,
                                 item_metadata_layers_dims=[12], combined_layers_dims=[16, 4],
                                 lr_scheduler_func=None, **kw)


def test_hybrid_head_with_blocks_is_built_saved_and_loaded(tmp_path):
    from collie_amd.hybrid import HybridPretrainedModel
    plain, deep = _hybrid(), _hybrid(combined_blocks=2)
    more = set(deep.state_dict()) - set(plain.state_dict())
    assert more == {f'combined_block_{i}.{n}.{p}' for i in range(2)
                    for n in ('norm', 'gated.gate', 'gated.up', 'back') for p in ('weight', 'bias')}
    assert deep.state_dict()['combined_block_1.gated.up.weight'].shape == (32, 16)
    deep.save_model(tmp_path / 'deep')
    loaded = HybridPretrainedModel(load_model_path=str(tmp_path / 'deep'))
    for k, v in deep.state_dict().items():
        assert torch.equal(v, loaded.state_dict()[k])
    copy = _hybrid()
    copy.load_from_hybrid_model(deep)
    assert len(copy.combined_blocks) == 2
    # a model saved before there were blocks
    plain.hparams.pop('combined_blocks')
    plain.save_model(tmp_path / 'plain')
    assert HybridPretrainedModel(load_model_path=str(tmp_path / 'plain')).combined_blocks == []
    with pytest.raises(ValueError, match='negative'):
        _hybrid(combined_blocks=-1)
    with pytest.raises(_lib.CollieHipError, match='no CPU fallback'):
        deep(torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.int64))
