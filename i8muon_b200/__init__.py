"""B200-native (sm_100a) Newton-Schulz orthogonalisation and Muon optimizer step.

Drop-in names of the reference package (src/i8muon/__init__.py:1-5):
``Muon``, ``muon_step``, ``CutlassNSInt8``, ``recommend_coefficients``; plus ``FusedAdamW``, a
companion for Muon's ``scalar_optimizer`` slot, and the layers whose gradients the two step on (``layers.py``).
"""
from .adamw import FusedAdamW
from .coefficients import recommend_coefficients
from .engine import CutlassNSInt8, check_status
from .layers import QuantisedActivation, layer_norm, linear, quantise_activation, restore_activation
from .optimizer import Muon, muon_step

__all__ = ["Muon", "muon_step", "CutlassNSInt8", "recommend_coefficients", "check_status", "FusedAdamW",
           "linear", "layer_norm", "quantise_activation", "restore_activation", "QuantisedActivation"]
