"""CPU tests of the hybrid model's residual blocks: copies between heads of different depth."""
import pytest
import torch


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


@pytest.mark.parametrize('named', [True, False])
@pytest.mark.parametrize('had,gets', [(2, 0), (0, 2), (3, 1), (1, 3)])
def test_a_model_becomes_the_copy_of_one_of_another_depth(had, gets, named):
    copy, source = _hybrid(combined_blocks=had), _hybrid(combined_blocks=gets)
    if not named:                           # hyper-parameters saved before there were blocks
        if gets:
            return
        source.hparams.pop('combined_blocks')
    copy.load_from_hybrid_model(source)
    assert len(copy.combined_blocks) == gets and copy.hparams.combined_blocks == gets
    state = source.state_dict()
    assert copy.state_dict().keys() == state.keys()
    for k, v in copy.state_dict().items():
        assert torch.equal(v, state[k])
