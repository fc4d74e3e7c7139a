"""settings.max_grad_norm reaches the optimizer of every training loop, without a GPU: the optimizers are replaced."""
import numpy as np
import pytest
import torch

from supernnova_amd import optim
from supernnova_amd.training import train_rnn
from supernnova_amd.utils import training_utils as tu
from test_host_logic import settings


class _Made(Exception):
    pass


def _record(model, **hyper):
    raise _Made(hyper)


@pytest.mark.parametrize("limit", [0.5, None, "absent"])
@pytest.mark.parametrize("loop", ["train_", "train_cyclic", "train_swag", "train_swag_finetune"])
def test_the_loops_pass_max_grad_norm_on(tmp_path, monkeypatch, loop, limit):
    monkeypatch.setattr(optim, "FusedSGD", _record)
    monkeypatch.setattr(optim, "FusedAdam", _record)
    st = settings(model="vanilla", use_cuda=False, batch_size=2, nb_epoch=1, monitor_interval=1, rnn_dir=str(tmp_path), learning_rate=5e-3,
                  pytorch_model_name="m", training_features_to_normalize=["f0"], arr_norm=np.zeros((1, 3)), cyclic=False, cyclic_phases=[1, 2, 3])
    if limit != "absent":
        st.max_grad_norm = limit
    torch.save(tu.get_model(st, 24).state_dict(), tmp_path / "pre.pt")
    st.swag_pretrained_path, st.swag_start_epoch = str(tmp_path / "pre.pt"), 0
    data = [(np.zeros((4, 24), np.float32), 0, "a")] * 4
    with pytest.raises(_Made) as made:
        getattr(train_rnn, loop)(st, data, data)
    assert made.value.args[0]["max_grad_norm"] == (None if limit == "absent" else limit)
