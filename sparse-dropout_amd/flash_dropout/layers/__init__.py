from .dropout_conv import DropoutConv2d
from .dropout_mm import DropoutMM
from .gated_mlp import GatedMLP
