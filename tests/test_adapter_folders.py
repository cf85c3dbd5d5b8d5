"""What the command line says of an adapter's folder that holds none."""
import json

import pytest
import torch

from foundry_b200 import cli
from foundry_b200.engine.adapters import AdapterError, AdapterStore
from foundry_b200.weights.safetensors_io import save_file
from test_adapter_store_failures import model_of, sites


class Engine:
    def enable_adapters(self, places, rank):
        self.held = AdapterStore(model_of(sites()), places, rank, torch.float32, "cpu")

    def load_adapter(self, *args):
        self.held.load(*args)


@pytest.mark.parametrize("tensors,what", [({}, "no tensors"), ({"a.o.lora_A.weight": torch.zeros(8), "a.o.lora_B.weight": torch.zeros(6, 1)}, "a.o"),
                                          ({"a.o.lora_A.weight": torch.zeros(169, 8), "a.o.lora_B.weight": torch.zeros(6, 169)}, "rank 169")])
def test_folders_without_an_adapter_that_fits(tmp_path, tensors, what):
    save_file(tensors, str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 6}))
    with pytest.raises(AdapterError, match=what):
        cli.load_adapter(Engine(), str(tmp_path))
