"""Caller-side glue with the reference's signatures: `render()` / `batchify_rays()` (core/trainer.py:64-145)
and the image losses / PSNR the trainer applies to the returned dict (core/trainer.py:8-61,353-380).

These are thin: ray-batch assembly and dict concatenation only; the chunks go to RayCaster (HIP kernels).
"""
import torch


def batchify_rays(rays_flat, chunk=1024 * 32, ray_caster=None, **kwargs):
    """core/trainer.py:64-79."""
    all_ret = {}
    n = rays_flat.shape[0]
    # A tensor kwarg with ONE row next to many rays is a value shared by every ray (render_path hands the frame's pose over
    # once, stride 0, instead of the reference's per-ray `reuse_input` expansion): it goes to every chunk whole.
    shared = {k for k, v in kwargs.items() if torch.is_tensor(v) and v.dim() > 0 and v.shape[0] == 1 and n > 1}
    if n <= chunk:
        # one chunk (every training step): the tensors go through WHOLE.  `x[0:chunk]` of a tensor that requires grad (the pose
        # layer's skts) is a SliceBackward node even when it selects everything: its backward is a zero fill of the full tensor + a
        # copy of the gradient into it (4.7 MB each way at 3072 rays, two launches on the launch floor at 384), for nothing.
        # And nothing to concatenate: torch.cat of a single tensor copies it.
        return dict(ray_caster(rays_flat, **kwargs))
    for i in range(0, n, chunk):
        batch_kwargs = {k: kwargs[k][i:i + chunk] if (torch.is_tensor(kwargs[k]) and k not in shared) else kwargs[k]
                        for k in kwargs}
        ret = ray_caster(rays_flat[i:i + chunk], **batch_kwargs)
        for k in ret:
            all_ret.setdefault(k, []).append(ret[k])
    return {k: torch.cat(all_ret[k], 0) for k in all_ret}


def render(H, W, focal, chunk=1024 * 32, rays=None, c2w=None, near=0., far=1., center=None, use_viewdirs=False,
           c2w_staticcam=None, **kwargs):
    """core/trainer.py:82-145 (the `rays` form: the reference's c2w form drops into pdb).
    near / far: numbers (one fused launch builds the ray batch) or tensors broadcastable to [N,1] (torch ops on the device, no
    host read).  c2w_staticcam (trainer.py:118-122): origins and directions of that second camera's full H x W image, view
    directions of the given rays."""
    from . import ops
    if rays is None:
        raise NotImplementedError("render() needs `rays`; build them with synth.camera_rays / the dataset")
    rays_o, rays_d = rays
    viewdirs = rays_d
    static = use_viewdirs and c2w_staticcam is not None
    if static:
        cam = torch.as_tensor(c2w_staticcam, dtype=torch.float32, device=rays_d.device)
        rb_s, _ = ops.gen_rays(H, W, focal, cam, (0, 0, W, H))               # get_rays(H, W, focal, c2w_staticcam), ray_utils.py:6-28
        rays_o, rays_d = rb_s[:, 0:3].reshape(H, W, 3), rb_s[:, 3:6].reshape(H, W, 3)
    sh = rays_d.shape
    rays_o = torch.reshape(rays_o, [-1, 3]).float()
    rays_d = torch.reshape(rays_d, [-1, 3]).float()
    # (an identity test `viewdirs is rays[1]` is never true for a [2,N,3] tensor: every unpack / index builds a new view object)
    plain = not torch.is_tensor(near) and not torch.is_tensor(far) and not static
    if plain:
        # (o, d, near, far [, d / |d|]) in one launch; the reference builds it with ones_like x2, norm, div and cat
        ray_batch = ops.make_ray_batch(rays_o, rays_d, near, far, use_viewdirs)
    else:
        ones = torch.ones_like(rays_d[..., :1])
        parts = [rays_o, rays_d, near * ones, far * ones]
        if use_viewdirs:
            vd = torch.reshape(viewdirs, [-1, 3]).float()
            parts.append(vd / torch.norm(vd, dim=-1, keepdim=True))
        ray_batch = torch.cat(parts, -1).contiguous()
    all_ret = batchify_rays(ray_batch, chunk, **kwargs)
    for k in all_ret:
        if all_ret[k].dim() >= 4:
            continue
        all_ret[k] = torch.reshape(all_ret[k], list(sh[:-1]) + list(all_ret[k].shape[1:]))
    return all_ret


@torch.no_grad()
def render_path(render_poses, hwf, chunk, render_kwargs, centers=None, kp=None, skts=None, cyls=None, bones=None,
                gt_imgs=None, bg_imgs=None, bg_indices=None, cams=None, subject_idxs=None, render_factor=0,
                white_bkgd=False, ret_acc=False, ext_scale=0.00035, base_bg=1.0):
    """run_nerf.render_path (run_nerf.py:28-145), same arguments and the same 5-tuple
    `(rgbs [F,H,W,3], disps [F,H,W,1], accs ([F,H,W,1] or []), valid_idxs, bboxes)`, with the frame-side work on the
    device: the 2-D boxes of ALL frames' projected cylinders come from one launch (k_cyl_bbox) and one small D2H copy
    before the first frame, rays of a box are generated by k_gen_rays, the pose is passed ONCE (stride-0, no per-ray
    replication), the background composite + scatter into the H*W image is k_assemble, and the finished frames stay on
    the device until the end of the call: ONE D2H copy for all of them (per 2 GB of frames).
    subject_idxs [F|1]: the subject of a frame, where the caster has adapters (RayCaster.set_adapters).
    H / W / focal may be per frame (sequences / arrays, as the h36m loader provides); kp [F|1,24,3], skts [F|1,24,4,4],
    cyls [F|1,5] (or None: derived from kp as kp_to_valid_rays does).  NaN disparities are zeroed (:139-140)."""
    from . import ops, synth
    import numpy as np
    H, W, focal = hwf
    is_scalar = lambda x: isinstance(x, (int, float, np.integer, np.floating))
    if render_factor != 0:      # run_nerf.py:37-48
        H = H // render_factor if is_scalar(H) else np.asarray(H) // render_factor
        W = W // render_factor if is_scalar(W) else np.asarray(W) // render_factor
        focal = focal / render_factor if is_scalar(focal) else np.asarray(focal).copy() / render_factor
        if centers is not None:
            centers = np.asarray(centers.cpu() if torch.is_tensor(centers) else centers).copy() / render_factor
    dev = kp.device
    pick = lambda x, i: None if x is None else (x[i % x.shape[0]:i % x.shape[0] + 1] if x.shape[0] > 1 else x)
    if cyls is None:
        cyls = torch.tensor(np.stack([synth.bounding_cylinder(k, ext_scale=ext_scale) for k in kp.cpu().numpy()]), device=dev)
    n_frames = len(render_poses)
    # ---- per-frame camera parameters on the host (inputs of the call), boxes of all frames in one launch
    hs, ws, fs, c2w_host, ctrs = [], [], [], [], []
    for i, c2w in enumerate(render_poses):
        hs.append(int(H) if is_scalar(H) else int(H[i]))
        ws.append(int(W) if is_scalar(W) else int(W[i]))
        f = focal if is_scalar(focal) else focal[i]                       # scalar or (fx, fy), ray_utils.py:8-11
        fs.append((float(f), float(f)) if is_scalar(f) or np.asarray(f).size < 2 else (float(f[0]), float(f[1])))
        c2w_host.append(np.asarray(c2w.cpu() if torch.is_tensor(c2w) else c2w, dtype=np.float32)[:3, :4])
        ctrs.append(None if centers is None else centers[i])
    if n_frames == 0:
        return np.zeros((0,)), np.zeros((0,)), ([] if not ret_acc else np.zeros((0,))), [], []
    off = np.array([[int(w * .5), int(h * .5)] if c is None else [int(c[0]), int(c[1])] for h, w, c in zip(hs, ws, ctrs)], np.int32)
    hwf64 = np.array([[h, w, f[0], f[1]] for h, w, f in zip(hs, ws, fs)], np.float64)
    c2w_all = torch.tensor(np.stack(c2w_host), device=dev)                # [F,3,4] fp32: the rays' camera; the boxes use it in double
    cyl_idx = torch.arange(n_frames, device=dev) % cyls.shape[0]
    boxes = ops.cyl_bbox(cyls.to(torch.float64)[cyl_idx].contiguous(), c2w_all.to(torch.float64).contiguous(),
                         torch.tensor(hwf64, device=dev), torch.tensor(off, device=dev)).cpu().numpy()     # the one sync up front
    kw = {k: v for k, v in render_kwargs.items() if k not in ("use_viewdirs",)}
    module = getattr(kw.get("ray_caster"), "module", kw.get("ray_caster"))
    adapted = subject_idxs is not None and getattr(module, "network", None) is not None and module.network.adapters() is not None
    valid_idxs, bboxes, packed, shapes = [], [], [], []
    out_rgb, out_disp, out_acc = [None] * n_frames, [None] * n_frames, [None] * n_frames
    pending_bytes = 0

    def flush():
        """every finished frame so far: one D2H copy, split on the host"""
        nonlocal packed, shapes, pending_bytes
        if not packed:
            return
        # straight into ONE pinned host buffer (a torch.cat first would hold every frame twice on the device), one sync
        total = sum(p.numel() for p in packed)
        host_t = torch.empty(total, dtype=torch.float32, pin_memory=True)
        o = 0
        for p in packed:
            host_t[o:o + p.numel()].copy_(p, non_blocking=True)
            o += p.numel()
        torch.cuda.current_stream(dev).synchronize()
        host = host_t.numpy()
        o = 0
        for i, h, w in shapes:
            npx = h * w
            out_rgb[i] = host[o:o + 3 * npx].reshape(h, w, 3); o += 3 * npx
            out_disp[i] = host[o:o + npx].reshape(h, w, 1); o += npx
            if ret_acc:
                out_acc[i] = host[o:o + npx].reshape(h, w, 1); o += npx
        packed, shapes, pending_bytes = [], [], 0

    for i in range(n_frames):
        h, w, f = hs[i], ws[i], fs[i]
        cyl_i = pick(cyls, i)
        x0, y0, x1, y1 = (int(v) for v in boxes[i])
        center = ctrs[i]
        rb, vidx = ops.gen_rays(h, w, f if f[0] != f[1] else f[0], c2w_all[i], (x0, y0, x1, y1), center=center)
        n = rb.shape[0]
        if bg_imgs is not None and not white_bkgd:
            bg = torch.as_tensor(bg_imgs[bg_indices[i] if bg_indices is not None else 0], dtype=torch.float32, device=dev)
            if bg.shape[0] != h or bg.shape[1] != w:
                bg = torch.nn.functional.interpolate(bg.permute(2, 0, 1)[None], size=(h, w), mode="bilinear",
                                                     align_corners=False)[0].permute(1, 2, 0)
            rgb_img = bg.reshape(h * w, 3).contiguous().clone()
        else:
            rgb_img = torch.full((h * w, 3), 1.0 if white_bkgd else 0.0, device=dev)
        disp_img = torch.zeros(h * w, device=dev)
        acc_img = torch.zeros(h * w, device=dev) if ret_acc else None
        if n > 0:
            cam_i = pick(cams, i)
            ret = batchify_rays(rb, chunk, kp_batch=pick(kp, i), skts=pick(skts, i),
                                cyls=cyl_i.expand(n, -1).contiguous(), bones=pick(bones, i),
                                cams=None if cam_i is None else cam_i.expand(n).contiguous(),
                                subject_idxs=pick(subject_idxs, i) if adapted else None, **kw)
            rgb_img, disp_img, acc_img = ops.assemble_frame(ret["rgb_map"], ret["acc_map"], ret["disp_map"], vidx, rgb_img,
                                                            want_acc=ret_acc)
        parts = [rgb_img.reshape(-1), torch.nan_to_num(disp_img, nan=0.0).reshape(-1)] + ([acc_img.reshape(-1)] if ret_acc else [])
        packed += parts
        shapes.append((i, h, w))
        pending_bytes += sum(p.numel() for p in parts) * 4
        valid_idxs.append(vidx)
        bboxes.append((np.array([x0, y0]), np.array([x1, y1])))
        if pending_bytes > (2 << 30):
            flush()
    flush()
    return np.stack(out_rgb, 0), np.stack(out_disp, 0), (np.stack(out_acc, 0) if ret_acc else []), valid_idxs, bboxes


def _reduce(d, reduction):
    return torch.mean(d) if reduction == "mean" else (torch.sum(d) if reduction == "sum" else d)


def img2mse(x, y, reduction="mean", to_yuv=False, scale_yuv=(0.1, 1.0, 1.0)):
    """core/trainer.py:10-25 (the YUV weighting is used by no shipped config)"""
    if to_yuv:
        raise NotImplementedError("to_yuv losses are not used by the shipped configs")
    return _reduce((x - y) ** 2, reduction)


def img2l1(x, y, reduction="mean", to_yuv=False, scale_yuv=(0.1, 1.0, 1.0)):
    """core/trainer.py:27-42"""
    if to_yuv:
        raise NotImplementedError("to_yuv losses are not used by the shipped configs")
    return _reduce((x - y).abs(), reduction)


def mse2psnr(x):
    return -10. * torch.log10(x)


def img2huber(x, y, reduction="mean", beta=0.1):
    """core/trainer.py:57-58"""
    return torch.nn.functional.smooth_l1_loss(x, y, reduction=reduction, beta=beta)


def nerf_loss(preds, target, bgs=1.0, loss_fn="MSE", coarse_weight=1.0, use_background=True, beta=0.1):
    """_compute_nerf_loss for the fine and coarse heads (core/trainer.py:353-380; get_loss_fn :146-156)."""
    if loss_fn not in ("MSE", "L1", "Huber"):
        raise NotImplementedError(loss_fn)
    fn = {"MSE": img2mse, "L1": img2l1, "Huber": lambda x, y: img2huber(x, y, beta=beta)}[loss_fn]
    def comp(rgb, acc):
        return rgb + (1. - acc)[..., None] * bgs if use_background else rgb
    pred = comp(preds["rgb_map"], preds["acc_map"])
    total = fn(pred, target)
    if "rgb0" in preds:
        total = total + coarse_weight * fn(comp(preds["rgb0"], preds["acc0"]), target)
    return total, pred
