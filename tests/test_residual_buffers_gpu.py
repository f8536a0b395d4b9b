"""What the residual GraphSAGE engine's layers share."""
import pytest
import torch

from grappa_b200.dataset import synthetic as S
from grappa_b200.graph_store import partition_from_global
from grappa_b200.models import get_model
from grappa_b200.trainer import FullGraphTrainer

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("bits", [16, 8])
def test_layers_share_one_gradient_buffer(bits):
    """Every layer's dY is written after the weight gradient that read the one before it, so one
    buffer, as large as the widest layer's, serves all."""
    g = S.build(S.SPECS["tiny"], DEV)
    own = partition_from_global(g, 1, 0, DEV)
    torch.manual_seed(0)
    model = get_model("sage", g.spec.feat_dim, g.spec.n_classes, num_hidden=64, num_layers=5, dropout=0.0,
                      activation="silu", norm="rms", residual=True)
    tr = FullGraphTrainer(model, own, act_bits=bits, use_cuda_graph=False)
    lay = tr.engine.lay
    assert len({s["dY"].untyped_storage().data_ptr() for s in lay}) == 1
    assert lay[0]["dY"].untyped_storage().nbytes() == max(s["dY"].numel() for s in lay) * 2
    for e in range(3):
        tr.train_epoch(e)
    tr.engine.check_errors()
    tr.close()
