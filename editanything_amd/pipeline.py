"""diffusers-style ControlNet (+inpaint) pipeline on the MI355X denoiser.

Call surface of `StableDiffusionControlNetInpaintPipeline.__call__`
(utils/stable_diffusion_controlnet_inpaint.py:1131-1703) and of the generation pipeline
`StableDiffusionControlNetPipeline2.__call__` (utils/stable_diffusion_controlnet.py:347-662):
same keyword names, same validation errors (`check_inputs` :792-979), `output_type` "pil" | "np" | "latent",
`callback(i, t, latents)`, `[uncond || cond]` CFG batch layout (:701), CPU-generator noise (:1005-1007),
4-channel vs 9-channel (SD2-inpainting) UNets, latent blending with `alignment_ratio` (:1647-1664),
list-valued `controlnet_conditioning_image` / `controlnet_conditioning_scale` for several ControlNets.

What is different underneath: the per-step work is `ControlledDenoiser.eps` (NHWC fp16 HIP kernels) plus ONE
fused CFG + sampler-step (+ inpaint blend) kernel, and the whole step is captured once in a HIP graph and
replayed (several hundred launches per step otherwise).  Samplers: DDIM in the reference LDM convention
(cldm/ddim_hacked.py, the parity sampler) and UniPC (`scheduler.UniPCMultistepScheduler`, the one the reference installs;
restated from the published algorithm because diffusers is absent -- parity unpinned): `pipe.scheduler =
UniPCMultistepScheduler.from_config(pipe.scheduler)` as in sam2image.py:42.
Text encoding is outside the hot path: pass `prompt_embeds` / `negative_prompt_embeds`, or give
the pipeline a `text_encoder` callable (list[str] -> [B, 77, ctx_dim]).
"""
import copy

import numpy as np
import torch
import torch.nn.functional as F

from . import host, ops
from .scheduler import DDIMScheduler, UniPCMultistepScheduler
from .unet import ControlledDenoiser


class StableDiffusionPipelineOutput:
    def __init__(self, images, nsfw_content_detected=None):
        self.images = images
        self.nsfw_content_detected = nsfw_content_detected

    def __iter__(self):
        return iter((self.images, self.nsfw_content_detected))


def loop_draw_count(nsteps, step_noise, mixing):
    """Random tensors (each of the latents' shape) the denoising loop consumes, in order: the mixing pipeline's re-noise in front
    of the steps (…inpaint.py:1968-1975), then per step the eta > 0 variance noise and -- every step but the last -- the mixing
    re-noise (:2039-2051)."""
    return (1 if mixing else 0) + (nsteps if step_noise else 0) + (nsteps - 1 if mixing else 0)


def randn_tensor(shape, generator=None, device=None, dtype=torch.float32):
    """diffusers.utils.randn_tensor semantics: a CPU generator draws on the CPU, then the sample moves."""
    gdev = generator.device.type if generator is not None else "cpu"
    if gdev == "cpu":
        return torch.randn(shape, generator=generator, dtype=dtype).to(device)
    return torch.randn(shape, generator=generator, device=device, dtype=dtype)


class _Call:
    """One pipeline call in flight: what `front` prepared, what `loop` left behind (attribute bag)."""


class StableDiffusionControlNetInpaintPipeline:
    vae_scale_factor = 8
    _guess_mode_cond_only = False   # the generation pipeline runs the ControlNet on the conditional half only in guess mode

    def __init__(self, vae, unet, controlnet, scheduler=None, text_encoder=None, tokenizer=None, device="cuda",
                 use_graph=True, denoiser_options=None):
        """denoiser_options: keyword arguments of `unet.ControlledDenoiser` (stream overlap, shared CFG prefix, twin launches)."""
        self.vae, self.unet = vae, unet
        self.controlnet = controlnet
        self.controlnets = list(controlnet) if isinstance(controlnet, (list, tuple)) else [controlnet]
        self.scheduler = scheduler or DDIMScheduler()
        self.text_encoder, self.tokenizer = text_encoder, tokenizer
        self.device = torch.device(device)
        self.denoiser = ControlledDenoiser(unet, self.controlnets, **(denoiser_options or {}))
        self.use_graph = use_graph
        self._graphs = {}       # (shape / mode key) -> {"st", "graph", "den"}: captured once, replayed by every later call
        self.trace = None       # set to a list: (phase name, torch.cuda.Event) marks are appended (bench.py --phases)

    def _mark(self, name):
        if self.trace is not None:
            e = torch.cuda.Event(enable_timing=True)
            e.record()
            self.trace.append((name, e))
            ops.profile_mark(name)

    # ---- no-op compatibility shims of the reference's pipeline object (sam2image.py:44-46, editany_lora.py:385-387)
    def to(self, device):
        return self

    def enable_xformers_memory_efficient_attention(self):
        pass

    def enable_model_cpu_offload(self):
        pass

    def load_textual_inversion(self, pretrained_model_name_or_path, token=None, **unused):
        """diffusers `TextualInversionLoaderMixin.load_textual_inversion` as the reference uses it (one local embedding
        file, editany_lora.py:733-735): a `.safetensors` / torch file holding either {token: vector(s)} or the
        Automatic1111 layout {"string_to_param": {"*": vectors}, "name": token}.  The token (and `token_1 .. token_{n-1}`
        for an n-vector embedding) is added to the tokenizer, the text encoder's embedding table is resized and the rows
        are written.  Needs the transformers tokenizer / text-encoder pair (models.load_text_encoder)."""
        if self.tokenizer is None or self.text_encoder is None or not hasattr(self.text_encoder, "resize_token_embeddings"):
            raise ValueError("load_textual_inversion needs a tokenizer and a transformers text encoder on the pipeline")
        from .convert import load_state_dict_file
        sd = load_state_dict_file(pretrained_model_name_or_path)
        if "string_to_param" in sd:
            loaded_token, emb = sd.get("name", token), sd["string_to_param"]["*"]
        else:
            if len(sd) != 1:
                raise ValueError("the embedding file must hold exactly one token")
            (loaded_token, emb), = sd.items()
        token = token if token is not None else loaded_token
        emb = emb if emb.ndim > 1 else emb[None]
        tokens = [token] + [f"{token}_{i}" for i in range(1, emb.shape[0])]
        vocab = self.tokenizer.get_vocab()
        if any(t in vocab for t in tokens):
            raise ValueError(f"Token {token} already in tokenizer vocabulary. Please choose a different token name or remove it.")
        self.tokenizer.add_tokens(tokens)
        ids = self.tokenizer.convert_tokens_to_ids(tokens)
        self.text_encoder.resize_token_embeddings(len(self.tokenizer))
        table = self.text_encoder.get_input_embeddings().weight
        with torch.no_grad():
            for i, row in zip(ids, emb):
                table[i] = row.to(table.dtype).to(table.device)
        return tokens

    # ------------------------------------------------------------------ input handling
    def check_inputs(self, prompt, image, mask_image, cond_images, height, width, callback_steps, negative_prompt,
                     prompt_embeds, negative_prompt_embeds, cond_scale):
        if height % 8 != 0 or width % 8 != 0:
            raise ValueError(f"`height` and `width` have to be divisible by 8 but are {height} and {width}.")
        if callback_steps is None or not isinstance(callback_steps, int) or callback_steps <= 0:
            raise ValueError(f"`callback_steps` has to be a positive integer but is {callback_steps}.")
        if prompt is not None and prompt_embeds is not None:
            raise ValueError("Cannot forward both `prompt` and `prompt_embeds`.")
        if prompt is None and prompt_embeds is None:
            raise ValueError("Provide either `prompt` or `prompt_embeds`.")
        if prompt is not None and not isinstance(prompt, (str, list)):
            raise ValueError(f"`prompt` has to be of type `str` or `list` but is {type(prompt)}")
        if negative_prompt is not None and negative_prompt_embeds is not None:
            raise ValueError("Cannot forward both `negative_prompt` and `negative_prompt_embeds`.")
        if prompt_embeds is not None and negative_prompt_embeds is not None and \
                prompt_embeds.shape != negative_prompt_embeds.shape:
            raise ValueError("`prompt_embeds` and `negative_prompt_embeds` must have the same shape.")
        n = len(self.controlnets)
        if not isinstance(self.controlnet, (list, tuple)):
            if not isinstance(cond_scale, float):
                raise TypeError("For single controlnet: `controlnet_conditioning_scale` must be type `float`.")
        else:
            if not isinstance(cond_images, list):
                raise TypeError("For multiple controlnets: `image` must be type `list`")
            if len(cond_images) != n:
                raise ValueError("For multiple controlnets: `image` must have the same length as the number of controlnets.")
            if isinstance(cond_scale, list) and len(cond_scale) != n:
                raise ValueError("For multiple controlnets: When `controlnet_conditioning_scale` is specified as `list`, it "
                                 "must have the same length as the number of controlnets")
        if (image is None) != (mask_image is None):
            raise ValueError("`image` and `mask_image` must be given together (inpainting) or both omitted.")
        from PIL import Image as _PIL
        if isinstance(image, torch.Tensor) and not isinstance(mask_image, torch.Tensor):
            raise TypeError("if `image` is a tensor, `mask_image` must also be a tensor")
        if isinstance(image, _PIL.Image) and not isinstance(mask_image, _PIL.Image):
            raise TypeError("if `image` is a PIL image, `mask_image` must also be a PIL image")
        if isinstance(image, torch.Tensor):          # …inpaint.py:903-963
            if image.ndim != 3 and image.ndim != 4:
                raise ValueError("`image` must have 3 or 4 dimensions")
            if mask_image.ndim not in (2, 3, 4):
                raise ValueError("`mask_image` must have 2, 3, or 4 dimensions")
            ib, ic, ih, iw = (1,) + tuple(image.shape) if image.ndim == 3 else tuple(image.shape)
            if mask_image.ndim == 2:
                mb, mc, mh, mw = (1, 1) + tuple(mask_image.shape)
            elif mask_image.ndim == 3:
                mb, mc, mh, mw = (mask_image.shape[0], 1) + tuple(mask_image.shape[1:])
            else:
                mb, mc, mh, mw = tuple(mask_image.shape)
            if ic != 3:
                raise ValueError("`image` must have 3 channels")
            if mc != 1:
                raise ValueError("`mask_image` must have 1 channel")
            if ib != mb:
                raise ValueError("`image` and `mask_image` mush have the same batch sizes")
            if ih != mh or iw != mw:
                raise ValueError("`image` and `mask_image` must have the same height and width dimensions")
            # value ranges: checked for host tensors only -- on device tensors each min()/max() is a blocking round trip
            # in front of the denoising loop (the reference pays it; a resident-input caller should not)
            if not image.is_cuda and (image.min() < -1 or image.max() > 1):
                raise ValueError("`image` should be in range [-1, 1]")
            if not mask_image.is_cuda and (mask_image.min() < 0 or mask_image.max() > 1):
                raise ValueError("`mask_image` should be in range [0, 1]")
        unet_in = getattr(getattr(self, "unet", None), "cfg", {}).get("in_channels", 4)
        if unet_in not in (4, 9):                    # :965-979: 4 latent channels, or 4 + 1 (mask) + 4 (masked image)
            raise ValueError(f"The config of `pipeline.unet` expects {unet_in} but received non inpainting latent "
                             f"channels: 4, mask channels: 1, and masked image channels: 4.")

    def _encode_text(self, prompts):
        """list[str] -> [B, L, ctx].  Two conventions: a plain callable `text_encoder(list[str])`, or the diffusers pair
        `tokenizer(...)` + `text_encoder(input_ids)[0]` (…inpaint.py:585-618: padded / truncated to `model_max_length`)."""
        if self.tokenizer is None:
            return self.text_encoder(prompts)
        ids = self.tokenizer(prompts, padding="max_length", max_length=self.tokenizer.model_max_length, truncation=True,
                             return_tensors="pt").input_ids
        return self.text_encoder(ids.to(getattr(self.text_encoder, "device", "cpu")))[0]

    def _encode_prompt(self, prompt, num_images_per_prompt, do_cfg, negative_prompt, prompt_embeds, negative_prompt_embeds):
        """…inpaint.py:551-703: -> [uncond || cond] embeddings, each repeated num_images_per_prompt times."""
        if prompt_embeds is None:
            if self.text_encoder is None:
                raise ValueError("This pipeline has no text encoder (outside the hot path): pass `prompt_embeds`.")
            prompts = [prompt] if isinstance(prompt, str) else list(prompt)
            prompt_embeds = self._encode_text(prompts)
            if do_cfg and negative_prompt_embeds is None:
                neg = negative_prompt if negative_prompt is not None else ""
                negs = [neg] * len(prompts) if isinstance(neg, str) else list(neg)
                if len(negs) != len(prompts):
                    raise ValueError("`negative_prompt` batch size must match `prompt`.")
                negative_prompt_embeds = self._encode_text(negs)
        prompt_embeds = prompt_embeds.to(self.device, torch.float32)
        b, L, _ = prompt_embeds.shape
        prompt_embeds = prompt_embeds.repeat(1, num_images_per_prompt, 1).view(b * num_images_per_prompt, L, -1)
        if do_cfg:
            if negative_prompt_embeds is None:
                raise ValueError("Classifier-free guidance needs `negative_prompt_embeds` (or a text encoder).")
            ne = negative_prompt_embeds.to(self.device, torch.float32)
            ne = ne.repeat(1, num_images_per_prompt, 1).view(b * num_images_per_prompt, L, -1)
            prompt_embeds = torch.cat([ne, prompt_embeds])
        return prompt_embeds

    def _cond_image_tensor(self, img, width, height):
        """A conditioning image argument of any accepted kind -> float tensor [b, 3, height, width] (tensors unscaled, PIL / uint8
        arrays LANCZOS-resized and scaled to [0, 1]): the first half of `_prepare_cond_image`, also what serving.merge_kwargs
        concatenates."""
        if not isinstance(img, torch.Tensor):
            if hasattr(img, "convert"):
                img = [img]
            if isinstance(img, np.ndarray):      # not a reference input kind: uint8 HWC / BHWC, treated like PIL
                arr = img[None] if img.ndim == 3 else img
                img = torch.from_numpy(arr.astype(np.float32) / 255.0).permute(0, 3, 1, 2)
            elif hasattr(img[0], "convert"):
                from PIL import Image as _PIL
                arr = np.concatenate([np.array(i.resize((width, height), resample=_PIL.LANCZOS))[None, :] for i in img], axis=0)
                img = torch.from_numpy(arr.astype(np.float32) / 255.0).permute(0, 3, 1, 2)
            else:
                img = torch.cat([i if i.ndim == 4 else i[None] for i in img], dim=0)
        img = img.float()
        if img.ndim == 3:
            img = img[None]
        if img.shape[-2:] != (height, width):
            img = F.interpolate(img, size=(height, width), mode="bilinear", align_corners=False)
        return img

    def _prepare_cond_image(self, img, width, height, batch, num_images_per_prompt, do_cfg):
        """prepare_controlnet_conditioning_image (…inpaint.py:328-388).  Tensors (or a list of tensors, concatenated)
        pass through unscaled -- the SAM id-map control is fed as float 0..255, sam2image.py:158-177; PIL images (or a
        list of them) are LANCZOS-resized to (width, height) and scaled to [0, 1].  One image is repeated for the whole
        batch, a batch of images `num_images_per_prompt` times each (repeat_interleave: [c0, c0, c1, c1], the order of
        the prompt embeddings)."""
        img = self._cond_image_tensor(img, width, height)
        repeat_by = batch if img.shape[0] == 1 else num_images_per_prompt
        img = img.repeat_interleave(repeat_by, dim=0)
        if img.shape[0] != batch:
            raise ValueError(f"controlnet conditioning image batch {img.shape[0]} does not match the effective batch size {batch}")
        img = img.to(self.device)
        return torch.cat([img] * 2) if do_cfg else img

    def prepare_latents(self, batch, channels, height, width, generator, latents=None):
        shape = (batch, channels, height // self.vae_scale_factor, width // self.vae_scale_factor)
        if isinstance(generator, list) and len(generator) != batch:
            raise ValueError(f"You have passed a list of generators of length {len(generator)}, but requested an "
                             f"effective batch size of {batch}.")
        if latents is None:
            if isinstance(generator, list):
                latents = torch.cat([randn_tensor((1,) + shape[1:], g, self.device) for g in generator])
            else:
                latents = randn_tensor(shape, generator, self.device)
        else:
            if tuple(latents.shape) != shape:
                raise ValueError(f"Unexpected latents shape, got {tuple(latents.shape)}, expected {shape}")
            latents = latents.to(self.device, torch.float32)
        return latents * self.scheduler.init_noise_sigma

    def _vae_noise(self, vae_noise, shape, generator):
        """Noise of the VAE posterior sample (`DiagonalGaussianDistribution.sample`, …inpaint.py:1079-1081).  Drawn from
        the call's generator right after the initial latents, as the reference does; `vae_noise=` lets a caller that
        batches several reference calls into one hand in the values those calls would have drawn (editany_lora.py)."""
        if vae_noise is not None:
            if tuple(vae_noise.shape) != tuple(shape):
                raise ValueError(f"Unexpected vae_noise shape, got {tuple(vae_noise.shape)}, expected {tuple(shape)}")
            return vae_noise.to(self.device, torch.float32)
        return randn_tensor(shape, generator if not isinstance(generator, list) else generator[0], self.device)

    def decode_latents(self, latents):
        """…inpaint.py:718-724 -> float32 NHWC numpy in [0, 1]."""
        img = self.vae.decode_nhwc(latents / self.vae.scale_factor)
        img = (img / 2 + 0.5).clamp(0, 1)
        return img.cpu().float().numpy()

    # ------------------------------------------------------------------ the step
    def _advance_inputs(self, st):
        """Self-advancing step (cached-graph path): the step's per-iteration inputs -- timestep, sampler coefficients, every
        ResBlock's time-embedding row -- are row `st["step"]` of tables that live in static buffers, gathered by a DEVICE
        index, which then advances (one launch, ops.gather_rows): all of it part of the captured graph, so a denoising
        loop is N back-to-back replays with no host-issued launch between them."""
        tab = st["tab"]
        pairs = [(tab["t"], st["t"]), (tab["coef"], st["coef"])] + list(zip(tab["embs"], st["embs"]))
        if st.get("unipc") is not None:
            pairs += [(tab["coefC"], st["unipc"]["coefC"]), (tab["coefP"], st["unipc"]["coefP"])]
        # ONE launch: every row gathered by the device index, which then advances (round 6: was four index_select + four to six
        # copy nodes + an add per step -- ~10 us per graph memcpy node)
        ops.gather_rows(pairs, st["step"], increment=1)

    def _step(self, st):
        if st.get("tab") is not None:
            self._advance_inputs(st)
        lat = st["lat"]
        if st["cfg"] and st["extra"] is None and self.denoiser.will_share_prefix(st["t"].shape[0], st.get("embs")):
            # the evaluation reads ONE copy of the CFG batch's identical halves: `cat([latents] * 2)` (…inpaint.py:1540-1547)
            # is never materialised (eps(cfg_single=True): x holds the conditional = unconditional rows once)
            eps = self.denoiser.eps(lat, st["t"], embs=st.get("embs"), cfg_halves=True, cfg_single=True)
        else:
            x2 = torch.cat([lat] * 2) if st["cfg"] else lat
            if st["extra"] is not None:                           # 9-ch inpaint UNet: latents || mask || masked latents
                x2 = torch.cat([x2, st["extra"]], dim=1)
            eps = self.denoiser.eps(x2, st["t"], embs=st.get("embs"), cfg_halves=bool(st["cfg"]))
        if st["cfg"]:
            e_u, e_c = eps.chunk(2)
        else:
            e_u, e_c = None, eps
        e_c, e_u = e_c.contiguous(), None if e_u is None else e_u.contiguous()
        if st.get("unipc") is None:
            ops.cfg_ddim_step(lat, e_c, e_u, st["coef"], noise=st["noise"], mask=st["blend_mask"], x_orig=st["x_orig"],
                              noise_orig=st["noise_orig"], x_prev=lat)
        else:
            # UniPC (scheduler.py): CFG + x0 prediction from the fused kernel, then corrector and predictor as two
            # linear combinations whose coefficients sit in device buffers (rows copied in per step)
            u = st["unipc"]
            ops.cfg_ddim_step(lat, e_c, e_u, st["coef"], x_prev=u["scratch"], pred_x0=u["m_t"])
            ops.lincomb([u["last"], u["m0"], u["m1"], u["m_t"], lat], u["coefC"], out=u["lat_c"])
            u["m1"].copy_(u["m0"])
            u["m0"].copy_(u["m_t"])
            u["last"].copy_(u["lat_c"])
            ops.lincomb([u["lat_c"], u["m0"], u["m1"]], u["coefP"], out=lat, mask=st["blend_mask"],
                        alt=(st["x_orig"], st["noise_orig"]))
        # (the sampler update writes the step's result straight into `lat`: both kernels are elementwise -- every element is read
        # before it is written by the same thread -- so no second buffer and no copy node)

    # ------------------------------------------------------------------ __call__
    @torch.no_grad()
    def __call__(self, *args, **kw):
        """The reference call (…inpaint.py:1131-1703) = the three stages below, back to back on the caller's stream.
        `serving.PipelinedRunner` runs the same three stages of CONSECUTIVE calls on two streams (front of call i+1 and
        back of call i-1 underneath the denoising loop of call i)."""
        call = self.front(*args, **kw)
        self.loop(call)
        return self.back(call)

    @torch.no_grad()
    def front(self, prompt=None, image=None, mask_image=None, controlnet_conditioning_image=None, height=None,
              width=None, num_inference_steps=50, guidance_scale=7.5, negative_prompt=None,
              num_images_per_prompt=1, eta=0.0, generator=None, latents=None, prompt_embeds=None,
              negative_prompt_embeds=None, output_type="pil", return_dict=True, callback=None, callback_steps=1,
              cross_attention_kwargs=None, controlnet_conditioning_scale=1.0, alignment_ratio=None,
              guess_mode=False, controlnet_conditioning_scale_map=None, vae_noise=None, alpha_weight=None, loop_noise=None,
              ref_image=None, ref_mask=None, ref_controlnet_conditioning_scale=1.0, ref_prompt=None,
              ref_prompt_embeds=None, attention_auto_machine_weight=1.0, gn_auto_machine_weight=1.0,
              style_fidelity=0.5, reference_attn=True, reference_adain=True, ref_scale=1.0, **unused):
        """Stage 1 of a call: validation, prompt / control / latent / inpaint-input preparation, VAE encode, and the
        per-call invariants of the denoiser (text K/V of every attention layer, ControlNet hint features, every step's
        time-embedding rows).  Touches NO state another call's `loop` reads: everything lands in tensors owned by the
        returned call object (the static buffers of the captured step are filled by `loop`).

        `ref_image` (+ `ref_mask`, `ref_prompt` or `ref_prompt_embeds`, ...): reference-only control,
        …inpaint.py:1163-1182, 1307-1605 (reference_only.py).  Write pass + read pass + sampler step are captured as one
        HIP graph per call (not cached across calls: banks, masks and module selection are per-call state)."""
        if controlnet_conditioning_image is None and "control_image" in unused:
            controlnet_conditioning_image = unused.pop("control_image")
        cond_images = controlnet_conditioning_image
        if not isinstance(cond_images, (list, tuple)):
            cond_images = [cond_images]
        ref = cond_images[0]
        if height is None or width is None:
            if isinstance(ref, torch.Tensor):
                height, width = height or ref.shape[-2], width or ref.shape[-1]
            else:
                arr = np.asarray(ref)
                height, width = height or arr.shape[0], width or arr.shape[1]
        self.check_inputs(prompt, image, mask_image, controlnet_conditioning_image, height, width, callback_steps,
                          negative_prompt, prompt_embeds, negative_prompt_embeds, controlnet_conditioning_scale)
        if prompt is not None:
            batch_size = 1 if isinstance(prompt, str) else len(prompt)
        else:
            batch_size = prompt_embeds.shape[0]
        do_cfg = guidance_scale > 1.0
        n_img = batch_size * num_images_per_prompt
        self._mark("start")
        embeds = self._encode_prompt(prompt, num_images_per_prompt, do_cfg, negative_prompt, prompt_embeds,
                                     negative_prompt_embeds)
        hints = [self._prepare_cond_image(ci, width, height, n_img, num_images_per_prompt, do_cfg) for ci in cond_images]
        n_out = len(self.unet.plan["input"]) + 1
        scales = controlnet_conditioning_scale
        if not isinstance(scales, (list, tuple)):
            scales = [scales] * len(self.controlnets)
        per_net = []
        for s in scales:
            if guess_mode:      # logspace ramp 0.1 .. 1 (utils/stable_diffusion_controlnet.py:777-783)
                ramp = torch.logspace(-1, 0, n_out).tolist()
                per_net.append([float(s) * r for r in ramp])
            else:
                per_net.append([float(s)] * n_out)
        nb_rows = 2 * n_img if do_cfg else n_img
        if controlnet_conditioning_scale_map is not None:
            # the reference multiplies EVERY net's scale by the map (utils/stable_diffusion_controlnet.py:490-495,
            # …inpaint.py:1874-1880); ControlNetModel2 then resizes it per level (bilinear, align_corners=True, :785-802)
            per_net = [self._scale_map_rows(controlnet_conditioning_scale_map, base, height, width, nb_rows)
                       for base in per_net]
        if guess_mode and do_cfg and self._guess_mode_cond_only:
            # generation pipeline, utils/stable_diffusion_controlnet.py:579-600: the ControlNet sees the conditional half
            # only and ZEROS are added to the unconditional half -> per-row scale 0 for the first n_img samples
            per_net = [self._zero_uncond_rows(base, height, width, n_img) for base in per_net]
        # a per-call copy: `loop` of the previous request may still be reading the scheduler's tables on another thread
        # (serving.PipelinedRunner); set_timesteps only REBINDS attributes, so a shallow copy isolates the call
        sch = copy.copy(self.scheduler)
        timesteps = sch.set_timesteps(num_inference_steps, eta=eta)
        lat = self.prepare_latents(n_img, 4, height, width, generator, latents)
        noise0 = lat.clone()
        unet_in = self.unet.cfg["in_channels"]
        extra = blend_mask = x_orig = None
        msk = None
        if image is not None:
            img = host.prepare_image(image).to(self.device)
            msk = host.prepare_mask_image(mask_image).to(self.device, torch.float32)
            if img.shape[-2:] != (height, width):
                img = F.interpolate(img, size=(height, width), mode="bilinear", align_corners=False)
                msk = F.interpolate(msk, size=(height, width), mode="nearest")
            h8, w8 = height // 8, width // 8
            if unet_in != 4:    # SD2-inpainting 9-channel UNet (…inpaint.py:1448-1468, 1550-1558)
                masked = img * (msk < 0.5)
                m_lat = F.interpolate(msk, size=(h8, w8))
                vnoise = self._vae_noise(vae_noise, (masked.shape[0], 4, h8, w8), generator)
                mi_lat = self.vae.encode(masked, vnoise)
                rep = n_img // m_lat.shape[0]
                m_lat, mi_lat = m_lat.repeat(rep, 1, 1, 1), mi_lat.repeat(n_img // mi_lat.shape[0], 1, 1, 1)
                extra = torch.cat([m_lat, mi_lat], dim=1)
                extra = torch.cat([extra] * 2) if do_cfg else extra
            else:               # 4-channel UNet: blend with the re-noised original (…inpaint.py:1469-1489, 1647-1664)
                vnoise = self._vae_noise(vae_noise, (img.shape[0], 4, h8, w8), generator)
                x_orig = self.vae.encode(img, vnoise)
                x_orig = x_orig.repeat(n_img // x_orig.shape[0], 1, 1, 1).contiguous()
                keep = 1 - F.interpolate(msk, size=(h8, w8), mode="nearest")
                keep = keep.repeat(n_img // keep.shape[0], 4, 1, 1).contiguous()
                blend_mask = (1 - keep).contiguous()         # 1 where the sample is generated
        c = _Call()
        c.ref_state = c.ref_ctx = None
        if ref_image is not None:
            c.ref_state, ref_den, ref_lat, ref_noise = self._prepare_reference(
                ref_image, ref_mask, ref_prompt, ref_prompt_embeds, ref_controlnet_conditioning_scale, hints, cond_images,
                width, height, n_img, num_images_per_prompt, do_cfg, generator, lat.shape, msk,
                unet_in, dict(style_fidelity=style_fidelity, ref_scale=ref_scale,
                              attention_auto_machine_weight=attention_auto_machine_weight,
                              gn_auto_machine_weight=gn_auto_machine_weight, reference_attn=reference_attn,
                              reference_adain=reference_adain), guess_mode)
            c.ref_ctx = dict(state=c.ref_state, den=ref_den, lat=ref_lat, noise=ref_noise, n_img=n_img, graph=None,
                             coef=torch.zeros(2, dtype=torch.float32, device=self.device))
        self._mark("inputs+vae_encode")
        unipc = isinstance(sch, UniPCMultistepScheduler)
        step_noise = eta > 0 and not unipc          # UniPC's step() takes no eta (prepare_extra_step_kwargs drops it)
        # alpha-weighted mixing (StableDiffusionControlNetInpaintMixingPipeline, …inpaint.py:1707-2088): its own blend
        # after every step (below) replaces the alignment_ratio blend of the plain pipeline and the final fill
        mixing = alpha_weight is not None and x_orig is not None
        if mixing and alignment_ratio is None:
            raise TypeError("the mixing pipeline compares `i < len(timesteps) * alignment_ratio`: pass alignment_ratio")
        in_loop_blend = x_orig is not None and alignment_ratio is not None and not mixing
        # One denoising step is captured ONCE per (shapes, mode) and replayed by every later call: the graph reads the
        # latents / text K,V / hint features / inpaint tensors from static buffers that `loop` overwrites in place.
        # Control scales are baked into the captured launches, so they are part of the key; per-pixel scale maps are
        # per-call tensors -> such calls capture afresh.
        gkey = None
        if self.use_graph and not step_noise and not in_loop_blend and c.ref_state is None and \
                all(not torch.is_tensor(v) for sc in per_net for v in sc):
            gkey = (type(sch).__name__, len(timesteps), n_img, height, width, do_cfg, unet_in, x_orig is not None, extra is not None, tuple(embeds.shape),
                    tuple(tuple(h.shape) for h in hints), tuple(tuple(sc) for sc in per_net))
        if unipc:
            c.coef_table, c.coef_c_table, c.coef_p_table = sch.coef_tables(guidance_scale, self.device)
        else:
            c.coef_table = sch.coef_table(guidance_scale, self.device)
        # the denoiser's per-call invariants (text K/V, hint features) and every step's time-embedding rows, as values
        c.invariants = self.denoiser.compute_invariants(embeds, hints)
        c.emb_tables = self.denoiser.time_embeddings(torch.as_tensor(timesteps.astype(np.int64), device=self.device))
        self._mark("prepare(hint,text kv)")
        c.sch, c.timesteps, c.lat, c.noise0, c.extra, c.blend_mask, c.x_orig = sch, timesteps, lat, noise0, extra, blend_mask, x_orig
        c.per_net, c.unipc, c.step_noise, c.mixing, c.in_loop_blend, c.gkey = per_net, unipc, step_noise, mixing, in_loop_blend, gkey
        c.do_cfg, c.n_img, c.generator, c.alignment_ratio, c.alpha_weight = do_cfg, n_img, generator, alignment_ratio, alpha_weight
        c.callback, c.callback_steps, c.output_type, c.return_dict = callback, callback_steps, output_type, return_dict
        # Every random draw of the LOOP is made here, in the order `loop` consumes it (one re-noise draw in front of the steps when
        # mixing; per step the eta > 0 variance noise, then the mixing re-noise): `loop` never touches the generator.  A call
        # draws front-then-loop from its generator whichever way it is run, so when serving.PipelinedRunner issues front(i + 1)
        # beside loop(i) -- possibly on the SAME generator object (torch.manual_seed returns the global one) -- request i + 1
        # still starts from the state request i's loop would have left: overlapped == sequential, bit for bit.
        # `loop_noise=`: those draws handed in (a sequence of `loop_draw_count` tensors of the latents' shape) -- what a caller that
        # batches several calls into one passes, like `latents=` / `vae_noise=` (serving.merge_kwargs).
        g0 = generator if not isinstance(generator, list) else generator[0]
        n_draws = loop_draw_count(len(timesteps), step_noise, mixing)
        if loop_noise is not None:
            if len(loop_noise) != n_draws or any(tuple(t.shape) != tuple(lat.shape) for t in loop_noise):
                raise ValueError(f"`loop_noise` must hold {n_draws} tensors of shape {tuple(lat.shape)}")
            c.loop_noise = [t.to(self.device, torch.float32) for t in loop_noise]
        else:
            c.loop_noise = [randn_tensor(lat.shape, g0, self.device) for _ in range(n_draws)]
        c.final = None
        return c

    def normalize_kwargs(self, kw):
        """The keyword form of a call as the BASE `front` sees it (subclasses fold their argument conventions in): what
        serving.predraw / merge_kwargs reason about."""
        return dict(kw)

    def loop_draws(self, num_inference_steps, eta, alpha_weight, has_image):
        """How many latents-shaped random tensors the loop of such a call consumes (`loop_draw_count`), by `front`'s own rules."""
        sch = copy.copy(self.scheduler)
        nsteps = len(sch.set_timesteps(num_inference_steps, eta=eta))
        step_noise = eta > 0 and not isinstance(sch, UniPCMultistepScheduler)
        mixing = alpha_weight is not None and has_image and self.unet.cfg["in_channels"] == 4
        return loop_draw_count(nsteps, step_noise, mixing)

    def has_graph(self, call):
        """True when `loop(call)` will replay an already captured step (nothing is captured, nothing allocated)."""
        return call.gkey is not None and call.gkey in self._graphs

    @torch.no_grad()
    def loop(self, c):
        """Stage 2: hand the call's tensors to the (static) buffers of the captured step, run the denoising steps, leave
        the final latents in `c.final` (a tensor the call owns)."""
        sch, timesteps = c.sch, c.timesteps
        nsteps = len(timesteps)
        draws = iter(c.loop_noise)          # pre-drawn by `front`, in this order
        lat, x_orig, extra, blend_mask = c.lat, c.x_orig, c.extra, c.blend_mask
        unipc, step_noise, mixing, in_loop_blend, gkey = c.unipc, c.step_noise, c.mixing, c.in_loop_blend, c.gkey
        ref_state, ref_ctx = c.ref_state, c.ref_ctx
        self.denoiser.only_mid_control = False
        ent = self._graphs.get(gkey) if gkey is not None else None
        nb = 2 * c.n_img if c.do_cfg else c.n_img
        if ent is not None:
            self.denoiser.install(c.invariants, c.per_net, static=ent["den"])
            st = ent["st"]
            st["lat"].copy_(lat)
            if extra is not None:
                st["extra"].copy_(extra)
            if x_orig is not None:
                st["x_orig"].copy_(x_orig)
                st["noise_orig"].copy_(c.noise0)
            graph = ent["graph"]
            if unipc:
                for k in ("m_t", "m0", "m1", "last", "lat_c"):
                    st["unipc"][k].zero_()
        else:
            self.denoiser.install(c.invariants, c.per_net)
            st = dict(lat=lat.contiguous(),
                      t=torch.zeros(nb, dtype=torch.long, device=self.device), coef=c.coef_table[0].clone(), cfg=c.do_cfg,
                      extra=extra, noise=None, blend_mask=None, x_orig=None if x_orig is None else x_orig.clone(),
                      noise_orig=c.noise0 if x_orig is not None else None)
            graph = None
            if unipc:
                z = lambda: torch.zeros_like(st["lat"])
                st["unipc"] = dict(m_t=z(), m0=z(), m1=z(), last=z(), lat_c=z(), scratch=z(),
                                   coefC=c.coef_c_table[0].clone(), coefP=c.coef_p_table[0].clone())
        # every step's time-embedding rows were computed in one shot; step i reads row i through the static [1, sum(Cout)] buffers
        emb_tables = c.emb_tables
        if st.get("embs") is None:
            st["embs"] = [tb[:1].clone() for tb in emb_tables]
        self_advance = gkey is not None      # cached-graph path: the captured step gathers its own row and counts (`_advance_inputs`)
        if self_advance:
            t_tab = torch.as_tensor(timesteps.astype(np.int64), device=self.device)
            new_tab = dict(t=t_tab, coef=c.coef_table, embs=list(emb_tables))
            if unipc:
                new_tab.update(coefC=c.coef_c_table, coefP=c.coef_p_table)
            if st.get("tab") is None:
                st["tab"] = {k: ([t.clone() for t in v] if isinstance(v, list) else v.clone()) for k, v in new_tab.items()}
                st["step"] = torch.zeros(1, dtype=torch.long, device=self.device)
            else:
                for k, v in new_tab.items():
                    for dst, src in zip(st["tab"][k] if isinstance(v, list) else [st["tab"][k]], v if isinstance(v, list) else [v]):
                        dst.copy_(src)
            st["step"].zero_()
        if mixing:   # …inpaint.py:1968-1975: the kept region starts from the re-noised original, the rest from pure noise
            self._mix_blend(st["lat"], x_orig, blend_mask, float(sch.alphas_cumprod[int(timesteps[0])]), 0.0, True, next(draws))
        for i in range(nsteps):
            if not self_advance:
                st["t"].fill_(int(timesteps[i]))
                st["coef"].copy_(c.coef_table[i])
                if unipc:
                    st["unipc"]["coefC"].copy_(c.coef_c_table[i])
                    st["unipc"]["coefP"].copy_(c.coef_p_table[i])
                for dst, tb in zip(st["embs"], emb_tables):
                    dst.copy_(tb[i:i + 1])
            st["noise"] = next(draws) if step_noise else None
            blend_now = in_loop_blend and i < nsteps * c.alignment_ratio and i + 1 < nsteps
            st["blend_mask"] = blend_mask if blend_now else None
            if ref_state is not None:
                # …inpaint.py:1562-1605: the reference latents, noised to this step's level, go through ControlNet + UNet
                # in write mode (features banked, output dropped); the real evaluation then reads the banks.  Both
                # passes + the sampler step are ONE captured graph per call (the banks, masks and module selection
                # are per-call state, so it is not cached across calls); the noise level comes from a static tensor.
                a_t = float(sch.alphas_cumprod[int(timesteps[i])])
                ref_ctx["coef"].copy_(torch.tensor([a_t ** 0.5, (1.0 - a_t) ** 0.5], dtype=torch.float32))
                if self.use_graph and not step_noise and not in_loop_blend and ref_state.graph_safe:
                    if ref_ctx["graph"] is None:
                        ref_ctx["graph"] = self._capture(st, ref_ctx)
                    ref_ctx["graph"].replay()
                else:
                    self._ref_step(st, ref_ctx)
            elif gkey is not None or (self.use_graph and not step_noise and not in_loop_blend):
                if graph is None:
                    graph = self._capture(st)
                    if gkey is not None:
                        # the entry owns everything the captured launches address: the static tensors, the denoiser's
                        # invariants and the scratch buffers of every stream of the step (ops.workspace_refs)
                        self._graphs[gkey] = dict(st=st, graph=graph, den=self.denoiser.static_state(),
                                                  scratch=ops.workspace_refs())
                graph.replay()
            else:
                self._step(st)
            if c.callback is not None and i % c.callback_steps == 0:
                c.callback(i, int(timesteps[i]), st["lat"])
            if mixing and i < nsteps - 1:     # …inpaint.py:2039-2051
                self._mix_blend(st["lat"], x_orig, blend_mask, float(sch.alphas_cumprod[int(timesteps[i + 1])]),
                                float(c.alpha_weight), i < nsteps * c.alignment_ratio, next(draws))
        c.final = st["lat"].clone()           # never hand out (or decode from) the captured step's static buffer
        self._mark("denoise loop")

    @torch.no_grad()
    def back(self, c):
        """Stage 3: final fill of the kept region, VAE decode, output conversion.  Reads only tensors the call owns."""
        lat = c.final
        if c.x_orig is not None and not c.mixing and (c.alignment_ratio is None or c.alignment_ratio == 1.0):
            lat = c.x_orig * (1 - c.blend_mask) + lat * c.blend_mask     # fill the kept region with the original
        if c.output_type == "latent":
            images = lat
        else:
            images = self.decode_latents(lat)
            if c.output_type == "pil":
                images = host.numpy_to_pil(images)
        self._mark("vae_decode")
        if not c.return_dict:
            return images, None
        return StableDiffusionPipelineOutput(images, None)

    def _prepare_reference(self, ref_image, ref_mask, ref_prompt, ref_prompt_embeds, ref_scale_cn, hints, cond_images, width,
                           height, n_img, nipp, do_cfg, generator, lat_shape, msk, unet_in, opts, guess_mode):
        """Everything the reference prepares once per `ref_image` call (…inpaint.py:1307-1315, 1348-1358, 1398-1425,
        1491-1534; prepare_ref_image / prepare_ref_latents stable_diffusion_reference.py:178-279): the reference prompt's
        embedding (no CFG), the reference image as [-1, 1] tensor and as the LAST ControlNet's conditioning image (the
        other nets keep the conditional half of theirs), its VAE latents, the noise it is re-noised with at every step, and
        a second denoiser state over the same networks for the write pass."""
        from .reference_only import ReferenceOnly
        from .unet import ControlledDenoiser
        if not self.controlnets:
            raise ValueError("reference-only control patches the last ControlNet: the pipeline has none")
        h8, w8 = height // 8, width // 8
        if ref_prompt_embeds is None:
            neg = ("longbody, lowres, bad anatomy, bad hands, missing fingers, extra digit, fewer digits, cropped, "
                   "worst quality, low quality")
            ref_embeds = self._encode_prompt(ref_prompt, nipp, False, neg, None, None)
        else:
            e = ref_prompt_embeds.to(self.device, torch.float32)
            ref_embeds = e.repeat(1, nipp, 1).view(e.shape[0] * nipp, e.shape[1], -1)
        if ref_embeds.shape[0] == 1 and n_img > 1:
            ref_embeds = ref_embeds.expand(n_img, -1, -1).contiguous()
        rmask = None
        if ref_mask is not None:
            rmask = F.interpolate(host.prepare_mask_image(ref_mask).float(), size=(h8, w8)).to(self.device)
        else:
            rmask = torch.ones(1, 1, h8, w8, device=self.device)
        # prepare_ref_image: RGB, LANCZOS to (width, height), [-1, 1]; one image is repeated over the batch
        rimg = ref_image
        if not isinstance(rimg, torch.Tensor):
            from PIL import Image as _PIL
            ims = [rimg] if hasattr(rimg, "convert") else list(rimg)
            if hasattr(ims[0], "convert"):
                arr = np.concatenate([np.array(i.convert("RGB").resize((width, height), resample=_PIL.LANCZOS))[None] for i in ims], 0)
                rimg = torch.from_numpy((arr.astype(np.float32) / 255.0 - 0.5) / 0.5).permute(0, 3, 1, 2)
            else:
                rimg = torch.cat(ims, dim=0)
        rimg = rimg.float()
        rimg = rimg.repeat_interleave(n_img if rimg.shape[0] == 1 else nipp, dim=0).to(self.device)
        ref_hint = self._prepare_cond_image(ref_image, width, height, n_img, nipp, False)
        ref_hints = [h[:h.shape[0] // 2] if do_cfg else h for h in hints]
        ref_hints[-1] = ref_hint
        # prepare_ref_latents: posterior sample from the call's generator (drawn after the inpaint latents, before the
        # re-noising noise -- the reference's order), scaled; then `noise = randn_tensor(latents.shape, generator)` :1528-1534
        g0 = generator if not isinstance(generator, list) else generator[0]
        vnoise = randn_tensor((rimg.shape[0], 4, h8, w8), g0, self.device)
        ref_lat = self.vae.encode(rimg, vnoise)
        if ref_lat.shape[0] < n_img:
            ref_lat = ref_lat.repeat(n_img // ref_lat.shape[0], 1, 1, 1)
        ref_noise = randn_tensor(tuple(lat_shape), generator, self.device) if not isinstance(generator, list) else \
            torch.cat([randn_tensor((1,) + tuple(lat_shape[1:]), g, self.device) for g in generator])
        scales = ref_scale_cn if isinstance(ref_scale_cn, (list, tuple)) else [ref_scale_cn] * len(self.controlnets)
        n_out = len(self.unet.plan["input"]) + 1
        per_net = []
        for sc in scales:
            ramp = torch.logspace(-1, 0, n_out).tolist() if guess_mode else [1.0] * n_out
            per_net.append([float(sc) * r for r in ramp])
        den = ControlledDenoiser(self.unet, self.controlnets)
        den.overlap = False
        den.prepare(ref_embeds, ref_hints, per_net)
        # the mask the AdaIN points restrict themselves to: `self.inpaint_mask = mask_image` after the pipeline's own
        # latent-resolution conversion (4-channel UNet: 1 - mask, :1488-1489; 9-channel: the mask itself)
        if msk is None:
            imask = torch.ones(1, 1, h8, w8, device=self.device)
        else:
            imask = (1 - F.interpolate(msk[:1], size=(h8, w8), mode="nearest")) if unet_in == 4 else msk[:1]
        state = ReferenceOnly(self.unet, self.controlnets[-1], n_img, do_cfg, rmask, imask, **opts)
        return state, den, ref_lat.contiguous(), ref_noise

    def _mix_blend(self, lat, x_orig, gen_mask, a_next, alpha, renoise_kept, noise):
        """In place, with proper = sqrt(a) * x_orig + sqrt(1 - a) * fresh noise (scheduler.add_noise at the next timestep):
            generated region (gen_mask = 1):  (1 - alpha) * lat + alpha * proper
            kept region      (gen_mask = 0):  proper if `renoise_kept` else lat
        One `ea_lincomb_f32` launch.  The reference draws the fresh noise with torch.randn_like on the device's global
        RNG (…inpaint.py:1975, 2041); here `noise` comes from the call's generator (drawn by `front`, in the loop's order), so a
        seeded call is reproducible."""
        c1, c2 = a_next ** 0.5, (1.0 - a_next) ** 0.5
        if renoise_kept:
            coef, alt = [1.0 - alpha, alpha * c1, alpha * c2, 0.0, 0.0, c1, c2], (x_orig, noise)
        else:
            coef, alt = [1.0 - alpha, alpha * c1, alpha * c2, 0.0, 0.0, 1.0, 0.0], (lat, None)
        out = ops.lincomb([lat, x_orig, noise], torch.tensor(coef, dtype=torch.float32, device=self.device),
                          mask=gen_mask, alt=alt)
        lat.copy_(out)

    def _ref_step(self, st, ref):
        """One denoising step under reference-only control: write pass over the noised reference latents, then the real
        step reading the banks (…inpaint.py:1562-1605)."""
        ref_xt = ref["coef"][0] * ref["lat"] + ref["coef"][1] * ref["noise"]
        ref["state"].begin("write")
        ref["den"].eps(ref_xt, st["t"][:ref["n_img"]])
        ref["state"].begin("read")
        self._step(st)
        ref["state"].end()

    def _capture(self, st, ref=None):
        """Warm up once on a side stream (restoring the latents), then capture ONE step into a HIP graph.  The warm-up
        also fills the per-call caches a capture could not (mask index lists, FFT plans).

        Round 6: while a HIP stream of NON-default priority exists in the process (serving.make_stream: the two-stream runner's
        low-priority side stream) some instantiations of the very same capture replay 1.3 - 2.6 x slower -- deterministically by
        instantiation count, eager launches unaffected (tools/probe_graph_lottery.py, profiles/r06_side_stream_priority.jsonl).  In
        that situation the step is instantiated three to five times, each timed over two replays on restored inputs, and the fastest
        kept (about one instantiation in three is slow, by 1.3 x and more; they can be consecutive)."""
        step = (lambda: self._ref_step(st, ref)) if ref is not None else (lambda: self._step(st))
        saved = st["lat"].clone()
        unipc_saved = {k: v.clone() for k, v in st["unipc"].items()} if st.get("unipc") is not None else None

        def restore():
            st["lat"].copy_(saved)
            if unipc_saved is not None:             # the multistep history a step pushed
                for k, v in unipc_saved.items():
                    st["unipc"][k].copy_(v)
            if st.get("tab") is not None:           # ... and the step index it advanced
                st["step"].zero_()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        restore()

        def instantiate():
            g = torch.cuda.CUDAGraph()
            with ops.graph_capture(g):
                step()
            restore()
            return g
        if not ops.nondefault_priority_streams() or ref is not None:      # (reference-only steps are captured per CALL: not worth 3 - 5 captures)
            return instantiate()
        # at least three instantiations, at most five; done once two of them sit within 10 % of the fastest seen (slow ones are
        # 1.3 x and more off, about one in three, and CAN be consecutive: two agreeing attempts alone prove nothing)
        tried = []
        for attempt in range(5):
            g = instantiate()
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            g.replay()                               # (first replay of an instantiation: uploads)
            e0.record()
            g.replay()
            g.replay()
            e1.record()
            torch.cuda.synchronize(self.device)
            restore()
            tried.append((e0.elapsed_time(e1), g))
            fastest = min(t for t, _ in tried)
            if attempt >= 2 and sum(1 for t, _ in tried if t <= 1.1 * fastest) >= 2:
                break
        return min(tried, key=lambda tg: tg[0])[1]

    def _level_sizes(self, height, width):
        """(h, w) of every ControlNet output: one per input block, plus the middle block."""
        sizes = []
        h8, w8 = height // 8, width // 8
        ds = 1
        for blk in self.unet.plan["input"]:
            if blk[0][0] == "down":
                ds *= 2
            sizes.append((h8 // ds, w8 // ds))
        sizes.append(sizes[-1])
        return sizes

    def _scale_map_rows(self, scale_map, base, height, width, nb):
        """ControlNetModel2 spatial scale map (utils/stable_diffusion_controlnet.py:785-802): per output level a bilinear
        (align_corners=True) resize of the [H, W] / [1, H, W] / [1, 1, H, W] map times the level's scalar scale -> one
        fp32 multiplier per output row (pixel), the same for every sample."""
        sm = torch.as_tensor(scale_map, dtype=torch.float32, device=self.device)
        sm = sm.reshape(1, 1, *sm.shape[-2:])
        rows = []
        for (hh, ww), b in zip(self._level_sizes(height, width), base):
            m = F.interpolate(sm, size=(hh, ww), mode="bilinear", align_corners=True).reshape(-1) * b
            rows.append(m.repeat(nb).contiguous())
        return rows

    def _zero_uncond_rows(self, base, height, width, n_img):
        rows = []
        for (hh, ww), b in zip(self._level_sizes(height, width), base):
            if torch.is_tensor(b):
                r = b.clone()
            else:
                r = torch.full((2 * n_img * hh * ww,), float(b), dtype=torch.float32, device=self.device)
            r[:n_img * hh * ww] = 0
            rows.append(r)
        return rows


class StableDiffusionControlNetInpaintMixingPipeline(StableDiffusionControlNetInpaintPipeline):
    """…inpaint.py:1707-2088: the same call with `alpha_weight` (default 0.5) -- after every step the generated region is
    pulled towards the re-noised original by alpha and the kept region is re-noised (first `alignment_ratio` of the
    steps) or left alone.  4-channel UNets only (the 9-channel inpainting UNet has no such blend, :2039)."""

    # the argument normalisation lives in `front`, the one entry both `__call__` and `serving.PipelinedRunner` go through
    def front(self, *args, alpha_weight=0.5, **kw):
        return super().front(*args, alpha_weight=alpha_weight, **kw)

    def normalize_kwargs(self, kw):
        return dict(kw, alpha_weight=kw.get("alpha_weight", 0.5))


class StableDiffusionControlNetPipeline(StableDiffusionControlNetInpaintPipeline):
    """Generation variant (sam2image.py:168-177 calls `pipe(prompt=..., image=control, ...)`): here `image` IS the
    ControlNet conditioning image, as in diffusers' StableDiffusionControlNetPipeline."""

    _guess_mode_cond_only = True    # utils/stable_diffusion_controlnet.py:579-600

    def front(self, prompt=None, image=None, **kw):
        if "controlnet_conditioning_image" not in kw:
            kw["controlnet_conditioning_image"] = image
            image = None
        return super().front(prompt=prompt, image=None, mask_image=None, **kw)

    def normalize_kwargs(self, kw):
        kw = dict(kw)
        image = kw.pop("image", None)
        kw.pop("mask_image", None)
        if "controlnet_conditioning_image" not in kw:
            kw["controlnet_conditioning_image"] = image
        return kw
