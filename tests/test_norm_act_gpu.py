"""norm_act (nnuzoo_amd/group_norm.py) takes the place of two module calls: what a caller could do with those - hooks registered for all
modules, forward-mode derivatives, vmap, second derivatives - gives the modules' results on token-major inputs, too."""
import pytest
import torch
from torch import nn

gpu = pytest.mark.gpu
ACTS = [nn.ReLU(inplace=True), nn.SiLU(), nn.LeakyReLU(0.2), nn.Identity()]
